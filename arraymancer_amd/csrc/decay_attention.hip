// Linear attention with a decay for each head: am_hip_decay_attention_*, am_hip_decay_attention_backward_*,
// am_hip_decay_attention_step_*.
//
// A head keeps a state S [dk, dv] and a token t with query q, key k and value v does
//     S <- e^g S + k^T v          o = scale * q S                        (g <= 0: the head's log_decay)
// Written out, o_i = scale * ( sum_{j <= i} e^{g (i - j)} (q_i . k_j) v_j + e^{g (i + 1)} q_i S_0 ).
//
// Its gradients are the same sum with other operands. With do the gradient of o and dS that of the last state:
//     dq_i = scale * ( sum_{j <= i} e^{g (i - j)} (do_i . v_j) k_j + e^{g (i + 1)} do_i S_0^T )
//            = the operator applied to (do, v, k) from the transposed state;
//     dv_j = sum_{i >= j} e^{g (i - j)} (k_j . q_i) scale do_i + e^{g (T - 1 - j)} k_j dS
//     dk_j = sum_{i >= j} e^{g (i - j)} (v_j . do_i) scale q_i + e^{g (T - 1 - j)} v_j dS^T
//            = the operator applied to (k, q, do) and to (v, do, q), walking from the last token to the first. The state of
//            that walk enters a token before it decays (e^{g n} instead of e^{g (n + 1)} for the n-th token), and what is
//            left of it behind the first token is the gradient of S_0.
// So one operator with four roles does everything; `Role` names its operands, and `after` is 1 for the walk forwards and 0
// for the walk backwards: e^{g (n + after)} is the n-th token's share of the first state, e^{g (N - after - n)} the n-th of
// N tokens' share in the last one.
#include "common.h"
#include "scratch.h"

namespace am {
namespace decay {

template <typename T> struct Operand { const T* p; int64_t b, t, h; int group; };   // head h reads h / group

// out = walk over the tokens with queries a, keys b, values c (dimensions da, da and dc)
template <typename T> struct Role {
  Operand<T> a, b, c;
  T* out; int64_t o_b, o_t, o_h;
  const T* s0; int64_t s0_b, s0_h, s0_r, s0_c;     // first state [da, dc], null: zeros
  T* s1; int64_t s1_b, s1_h, s1_r, s1_c;           // last state, null: not wanted
  T scale_a, scale_b;                // of the queries, of the keys
  int da, dc;
  const T* log_decay;
  const int64_t* lengths;
  int64_t batch, tokens, heads;      // heads: of the state and of log_decay
};

__device__ __forceinline__ float dev_exp(float v) { return expf(v); }
__device__ __forceinline__ double dev_exp(double v) { return exp(v); }
// e^{g n}; e^0 also where g is -infinity
template <typename T> __device__ __forceinline__ T power(T g, int64_t n) { return n == 0 ? (T)1 : dev_exp(g * (T)n); }

template <typename T> struct Mma;
template <> struct Mma<float> {
  typedef float acc_t __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ acc_t mma(float a, float b, acc_t c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }
  // the operand row that lane % 16 = r brings, so that register i of lane group g holds row 4 g + i of the result
  static __device__ __forceinline__ int row(int r) { return r; }
};
template <> struct Mma<double> {
  typedef double acc_t __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ acc_t mma(double a, double b, acc_t c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
  // (this instruction's result has row 4 i + g there)
  static __device__ __forceinline__ int row(int r) { return 4 * (r & 3) + (r >> 2); }
};

// ---- chunks of 32 tokens on the matrix cores ---------------------------------------------------------------------------
//
// For the tokens of a chunk, i and j counted within it, and the state S in front of it,
//     o_i = sum_{j <= i} A_ij c_j + e^{g (i + after)} a_i S      A_ij = e^{g (i - j)} (a_i . b_j)
//     S <- e^{g N} S + sum_j e^{g (N - after - j)} b_j^T c_j
// so a chunk is four products: a b^T (32 x 32), A c, a S and b^T c. A workgroup of four wavefronts walks the chunks of one
// head, a wavefront owning 16 columns of S and of o for all da rows, as accumulators that never leave its registers:
//   - the 16 x 16 x 4 product leaves four consecutive rows of its result in a lane, and the sum over k may take its k in any
//     order that both operands share: register i of S's tile is the right operand of the i-th of four instructions whose k
//     are the rows 4 g + i. So S enters a S as it stands.
//   - a b^T is computed transposed, so that a lane's four values lie next to each other in a row of A in LDS; the three
//     tiles on and under the diagonal go to three wavefronts.
//   - c is read straight into the layout of a right operand, which A c and b^T c share.
// a and b go through LDS in rows padded by 16 bytes; the next chunk's are on their way in registers meanwhile.
// All exponents of e^g are differences that the mask leaves >= 0, so nothing overflows however long the text.
//
// Where the heads alone do not fill the device, the tokens are cut into segments: `segment_sums` adds up each segment's
// share of the state, `segment_states` carries them from segment to segment, and `chunks` starts every segment from its own.
constexpr int64_t kMostDim = 256;
constexpr int kChunk = 32;
constexpr int kCols = 64;      // columns of a workgroup
constexpr int kLds = 160 * 1024;

template <typename T> struct Plan {
  T* states;                   // [batch * heads][slots][da][dc]: the state in front of each part; null: one segment
  int segments, slices;
  int parts, slots;            // parts of a segment; slots = parts * (segments - 1) + 1, one in front of every part but the last segment's later ones
  int64_t seg_tokens, part_tokens;   // multiples of kChunk, seg_tokens = parts * part_tokens
  int groups;                  // batch * heads
};

// The n <= 32 tokens of a chunk as a buffer: the hardware adds a lane's 32-bit offset to a uniform base, and what lies outside
// the buffer reads as 0 and is not written, so a short chunk needs neither branches nor clamped addresses. Token `row` lies
// `row * step` elements behind the chunk's first one; with a negative step the base is the last token's address, and tokens
// behind the last get offsets that wrap around, out of the buffer. Needs 32 steps to lie within 2^31 bytes.
struct Chunk { __amdgpu_buffer_rsrc_t rsrc; uint32_t first; };    // first: offset of the chunk's first token
template <typename T> __device__ __forceinline__ Chunk chunk_of(const T* p, int64_t step, int n, int width) {
  const T* base = step < 0 ? p + (n - 1) * step : p;
  const int reach = (n - 1) * (int)(step < 0 ? -step : step);
  Chunk c;
  c.rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)base, 0, (reach + width) * (int)sizeof(T), 0x00020000);
  c.first = step < 0 ? (uint32_t)(reach * (int)sizeof(T)) : 0u;
  return c;
}
__device__ __forceinline__ void get(const Chunk& c, uint32_t off, float& v) { v = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(c.rsrc, (int)off, 0, 0)); }
__device__ __forceinline__ void get(const Chunk& c, uint32_t off, double& v) { v = __builtin_bit_cast(double, __builtin_amdgcn_raw_buffer_load_b64(c.rsrc, (int)off, 0, 0)); }
__device__ __forceinline__ void put(const Chunk& c, uint32_t off, float v) { __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), c.rsrc, (int)off, 0, 0); }
__device__ __forceinline__ void put(const Chunk& c, uint32_t off, double v) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, v), c.rsrc, (int)off, 0, 0);
}

// The rows of up to 32 tokens of an operand, as 16-byte vectors in registers on their way to LDS. Every lane always loads (a
// load under a branch would have to be waited for before the next one). FAST: rows are whole vectors and the chunks buffers;
// else element by element from clamped addresses. What lies outside becomes 0 on the way into LDS.
template <typename T, int DA, bool FAST> struct Tile {
  static constexpr int V = 16 / (int)sizeof(T), PER_ROW = DA / V, NV = kChunk * PER_ROW / 256;
  static constexpr bool EVEN = 256 % PER_ROW == 0;       // vector u of a lane lies whole rows behind its first
  static constexpr int NO = EVEN ? 1 : NV;
  typedef T vec_t __attribute__((ext_vector_type(V)));
  static constexpr int PITCH = DA + V;
  vec_t v[NV];
  uint32_t off[NO];                                      // of a lane's vectors behind the chunk's first token

  __device__ __forceinline__ void prepare(int64_t step, int da) {
    if constexpr (FAST) {
#pragma unroll
      for (int u = 0; u < NO; ++u) {
        const int f = (int)threadIdx.x + u * 256, row = f / PER_ROW, c = (f - row * PER_ROW) * V;
        off[u] = (uint32_t)((row * (int)step + c) * (int)sizeof(T));
      }
    }
  }
  // p: the first token's row; step: to the next token; n >= 1 tokens
  __device__ __forceinline__ void load(const T* p, int64_t step, int n, int da) {
    if constexpr (FAST) {
      const Chunk k = chunk_of(p, step, n, da);
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const uint32_t o = EVEN ? off[0] + (k.first + (uint32_t)(u * (256 / PER_ROW) * (int)step * (int)sizeof(T))) : off[u % NO] + k.first;
        v[u] = __builtin_bit_cast(vec_t, __builtin_amdgcn_raw_buffer_load_b128(k.rsrc, (int)o, 0, 0));
      }
    } else {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int f = (int)threadIdx.x + u * 256;
        int row = f / PER_ROW, c = (f - row * PER_ROW) * V;
        row = row < n ? row : n - 1;
        const T* q = p + row * step;
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] = q[c + e < da ? c + e : da - 1];
      }
    }
  }
  __device__ __forceinline__ void store(T* lds, int n, int da) const {
    const bool all = n == kChunk && da == DA;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int f = (int)threadIdx.x + u * 256, row = f / PER_ROW, c = (f - row * PER_ROW) * V;
      vec_t w = v[u];
      if (!all) {
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = (row < n && c + (FAST ? 0 : e) < da) ? w[e] : (T)0;
      }
      *(vec_t*)(lds + row * PITCH + c) = w;
    }
  }
};

// Four neighbouring elements of LDS.
template <typename T> __device__ __forceinline__ void four(const T* lds, T (&out)[4]) {
  constexpr int V = 16 / (int)sizeof(T);
  typedef T vec_t __attribute__((ext_vector_type(V)));
#pragma unroll
  for (int i = 0; i < 4; i += V) {
    const vec_t w = *(const vec_t*)(lds + i);
#pragma unroll
    for (int e = 0; e < V; ++e) out[i + e] = w[e];
  }
}

// Nothing moves across here: the LDS reads of the next step stay in front of the matrix instructions of this one. Left alone,
// the scheduler puts every read right in front of its use, and the wavefront waits for LDS in every step.
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// What a workgroup works on. The slices of one (head, segment) read the same a and b: they get ids that are equal modulo
// the eight dies, whose L2 they share.
struct Work { int slice, segment, group; bool live; };
template <typename T> __device__ __forceinline__ Work work_of(const Plan<T>& pl, int segments) {
  const unsigned id = blockIdx.x, rest = id >> 3;
  Work w;
  w.slice = (int)(rest % (unsigned)pl.slices);
  const unsigned item = (rest / (unsigned)pl.slices) * 8 + (id & 7);
  w.segment = (int)(item % (unsigned)segments);
  w.group = (int)(item / (unsigned)segments);
  w.live = w.group < pl.groups;
  return w;
}

template <typename T> __device__ __forceinline__ int64_t length_of(const Role<T>& p, int64_t b) {
  if (!p.lengths) return p.tokens;
  const int64_t l = p.lengths[b];
  return l < 0 ? 0 : (l < p.tokens ? l : p.tokens);
}

// One wavefront's share of a chunk's sum over the tokens: S <- e^{g N} S + b^T (w c), c given weighted.
template <typename T, int DA>
__device__ __forceinline__ void add_tokens(typename Mma<T>::acc_t (&S)[DA / 16], const T* sB, const T (&wc)[2][4], T lam, int pr, int g) {
  constexpr int PITCH = DA + 16 / (int)sizeof(T);
#pragma unroll
  for (int kt = 0; kt < DA / 16; ++kt) {
    S[kt] *= lam;
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S[kt] = Mma<T>::mma(sB[(16 * jt + 4 * g + r) * PITCH + 16 * kt + pr], wc[jt][r], S[kt]);
  }
}

// c of a chunk of n >= 1 tokens, in the layout of a right operand: register r of tile jt is token 16 jt + 4 g + r, in column
// `col`. `take` makes tokens behind the n-th 0.
template <typename T, bool FAST>
__device__ __forceinline__ void load_c(T (&c)[2][4], const T* p, int64_t step, int n, int g, int col, int width) {
  if constexpr (FAST) {
    const Chunk k = chunk_of(p, step, n, width);
    const uint32_t off = (uint32_t)((4 * g * (int)step + col) * (int)sizeof(T));
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) get(k, off + (k.first + (uint32_t)((16 * jt + r) * (int)step * (int)sizeof(T))), c[jt][r]);
  } else {
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = 16 * jt + 4 * g + r;
        c[jt][r] = p[(j < n ? j : n - 1) * step + col];
      }
  }
}
template <typename T>
__device__ __forceinline__ void take(T (&c)[2][4], const T (&from)[2][4], int n, int g) {
  if (n == kChunk) {
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) c[jt][r] = from[jt][r];
    return;
  }
#pragma unroll
  for (int jt = 0; jt < 2; ++jt)
#pragma unroll
    for (int r = 0; r < 4; ++r) c[jt][r] = 16 * jt + 4 * g + r < n ? from[jt][r] : (T)0;
}

// scale * e^{g (n - after - j)} of this lane's tokens
template <typename T>
__device__ __forceinline__ void weights(T (&w)[2][4], T scale, T ld, int n, int after, int g) {
#pragma unroll
  for (int jt = 0; jt < 2; ++jt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int e = n - after - (16 * jt + 4 * g + r);
      w[jt][r] = scale * power(ld, (int64_t)(e > 0 ? e : 0));
    }
}

#ifndef WPE
#define WPE 2
#endif
template <typename T, int DA, bool BACK, bool FAST>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? WPE : 1) void chunks(Role<T> p, Plan<T> pl) {
  typedef typename Mma<T>::acc_t acc_t;
  typedef Tile<T, DA, FAST> tile_t;
  constexpr int KT = DA / 16, V = tile_t::V, PITCH = tile_t::PITCH, APITCH = kChunk + V;
  constexpr int after = BACK ? 0 : 1;
  constexpr int BUFS = (4 * kChunk * PITCH + kChunk * APITCH) * (int)sizeof(T) <= kLds ? 2 : 1;
  __shared__ __attribute__((aligned(16))) T bufs[BUFS][2][kChunk * PITCH];
  __shared__ __attribute__((aligned(16))) T sA[kChunk * APITCH];
  const Work w = work_of(pl, pl.segments);
  if (!w.live) return;
  const int64_t b = w.group / (int)p.heads;
  const int h = (int)(w.group - b * p.heads);
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, lr = lane & 15, pr = Mma<T>::row(lr);
  const int col = w.slice * kCols + wave * 16 + lr;
  const bool live = col < p.dc;
  const int64_t n = length_of(p, b);
  const int64_t lo = w.segment * pl.seg_tokens;
  int64_t hi = lo + pl.seg_tokens;
  if (hi > p.tokens) hi = p.tokens;
  const int64_t end = hi < n ? hi : n;                      // local tokens lo .. end of the walk
  // local token i is token i, or n - 1 - i
  const int64_t first = BACK ? n - 1 - lo : lo, dir = BACK ? -1 : 1;
  const T* pa = p.a.p + b * p.a.b + (h / p.a.group) * p.a.h + first * p.a.t;
  const T* pb = p.b.p + b * p.b.b + (h / p.b.group) * p.b.h + first * p.b.t;
  const T* pc = p.c.p + b * p.c.b + (h / p.c.group) * p.c.h + first * p.c.t;
  const int ccol = live ? col : p.dc - 1;
  T* po = p.out + b * p.o_b + h * p.o_h;
  const int64_t ta = dir * p.a.t, tb = dir * p.b.t, tc = dir * p.c.t;

  acc_t S[KT];
  const T* s0 = pl.states ? pl.states + ((int64_t)w.group * pl.slots + w.segment * pl.parts) * p.da * p.dc : (p.s0 ? p.s0 + b * p.s0_b + h * p.s0_h : nullptr);
  const int64_t s0_r = pl.states ? p.dc : p.s0_r, s0_c = pl.states ? 1 : p.s0_c;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * kt + 4 * g + r;
      S[kt][r] = (s0 && live && d < p.da) ? s0[d * s0_r + col * s0_c] : (T)0;
    }
  const T ld = p.log_decay[h];
  T reach[2][4], mask[2][4], wt[2][4];
#pragma unroll
  for (int it = 0; it < 2; ++it)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      reach[it][r] = p.scale_a * power(ld, (int64_t)(16 * it + 4 * g + r + after));
      const int apart = 16 * it + lr - 4 * g - r;          // i - j of tile distance `it`, transposed
      mask[it][r] = apart >= 0 ? p.scale_a * p.scale_b * power(ld, (int64_t)apart) : (T)0;
    }
  weights(wt, p.scale_b, ld, kChunk, after, g);
  T lam = power(ld, (int64_t)kChunk);

  tile_t a, k;
  T c[2][4], cn[2][4];
  a.prepare(ta, p.da);
  k.prepare(tb, p.da);
  const int64_t to = dir * p.o_t;
  const int64_t total = end - lo;
  if (total > 0) {
    const int m = total < kChunk ? (int)total : kChunk;
    a.load(pa, ta, m, p.da);
    k.load(pb, tb, m, p.da);
    load_c<T, FAST>(cn, pc, tc, m, g, ccol, p.dc);
    a.store(bufs[0][0], m, p.da);
    k.store(bufs[0][1], m, p.da);
  }
  int turn = 0;
  for (int64_t at = 0; at < total; at += kChunk) {
    const int64_t next = at + kChunk;
    const int m = total - at < kChunk ? (int)(total - at) : kChunk;
    const int mn = total - next < kChunk ? (int)(total - next) : kChunk;
    const T* sQ = bufs[turn][0];
    const T* sB = bufs[turn][1];
    take(c, cn, m, g);
    __syncthreads();
    if (next < total) {
      a.load(pa + next * ta, ta, mn, p.da);
      k.load(pb + next * tb, tb, mn, p.da);
      load_c<T, FAST>(cn, pc + next * tc, tc, mn, g, ccol, p.dc);
    }
    if (wave < 3) {                                         // tiles (0, 0), (1, 0), (1, 1) of A
      const int it = wave ? 1 : 0, jt = wave == 2 ? 1 : 0;
      acc_t t = (acc_t)((T)0);
      const T* px = sB + (16 * jt + pr) * PITCH + 4 * g;
      const T* py = sQ + (16 * it + lr) * PITCH + 4 * g;
      T x[2][4], y[2][4];
      four(px, x[0]);
      four(py, y[0]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if (kt + 1 < KT) {
          four(px + 16 * (kt + 1), x[(kt + 1) & 1]);
          four(py + 16 * (kt + 1), y[(kt + 1) & 1]);
        }
        pin();
#pragma unroll
        for (int r = 0; r < 4; ++r) t = Mma<T>::mma(x[kt & 1][r], y[kt & 1][r], t);
        pin();
      }
      T* q = sA + (16 * it + lr) * APITCH + 16 * jt + 4 * g;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool under = it > jt || lr >= 4 * g + r;
        q[r] = under ? t[r] * (it > jt ? mask[1][r] : mask[0][r]) : (T)0;
      }
    }
    acc_t o[2];
    {
      const T* px = sQ + pr * PITCH + 4 * g;
      T x[2][2][4];
      o[0] = o[1] = (acc_t)((T)0);
      four(px, x[0][0]);
      four(px + 16 * PITCH, x[0][1]);
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        if (kt + 1 < KT) {
          four(px + 16 * (kt + 1), x[(kt + 1) & 1][0]);
          four(px + 16 * PITCH + 16 * (kt + 1), x[(kt + 1) & 1][1]);
        }
        pin();
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          o[0] = Mma<T>::mma(x[kt & 1][0][r], S[kt][r], o[0]);
          o[1] = Mma<T>::mma(x[kt & 1][1][r], S[kt][r], o[1]);
        }
        pin();
      }
    }
#pragma unroll
    for (int it = 0; it < 2; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[it][r] *= reach[it][r];
    __syncthreads();
    {
      const T* px = sA + pr * APITCH + 4 * g;
      T x[3][4];
      four(px, x[0]);
      four(px + 16 * APITCH, x[1]);
      four(px + 16 * APITCH + 16, x[2]);
      pin();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        o[0] = Mma<T>::mma(x[0][r], c[0][r], o[0]);
        o[1] = Mma<T>::mma(x[1][r], c[0][r], o[1]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) o[1] = Mma<T>::mma(x[2][r], c[1][r], o[1]);
    }
    if (m < kChunk) { weights(wt, p.scale_b, ld, m, after, g); lam = power(ld, (int64_t)m); }
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) c[jt][r] *= wt[jt][r];
    add_tokens<T, DA>(S, sB, c, lam, pr, g);
    if (live) {
      T* q = po + (first + dir * at) * p.o_t;
      if constexpr (FAST) {
        const Chunk k = chunk_of(q, to, m, p.dc);
        const uint32_t off = (uint32_t)((4 * g * (int)to + col) * (int)sizeof(T));
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int r = 0; r < 4; ++r) put(k, off + (k.first + (uint32_t)((16 * it + r) * (int)to * (int)sizeof(T))), o[it][r]);
      } else {
#pragma unroll
        for (int it = 0; it < 2; ++it)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 16 * it + 4 * g + r;
            if (i < m) q[i * to + col] = o[it][r];
          }
      }
    }
    // the next chunk into LDS: into the other buffer, or (where two do not fit) behind a barrier
    if constexpr (BUFS == 2) turn ^= 1;
    else __syncthreads();
    if (next < total) {
      a.store(bufs[turn][0], mn, p.da);
      k.store(bufs[turn][1], mn, p.da);
    }
  }
  if (live) {                                               // behind the sequence
    for (int64_t t = (lo > n ? lo : n) + g; t < hi; t += 4) po[t * p.o_t + col] = (T)0;
  }
  if (p.s1 && w.segment == pl.segments - 1 && live) {
    T* s1 = p.s1 + b * p.s1_b + h * p.s1_h + col * p.s1_c;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 16 * kt + 4 * g + r;
        if (d < p.da) s1[d * p.s1_r] = S[kt][r];
      }
  }
}

// The share of a part (of all segments but the last) in the state behind it, into the slot behind the part's own.
template <typename T, int DA, bool BACK, bool FAST>
__global__ __launch_bounds__(256) void segment_sums(Role<T> p, Plan<T> pl) {
  typedef typename Mma<T>::acc_t acc_t;
  typedef Tile<T, DA, FAST> tile_t;
  constexpr int KT = DA / 16, PITCH = tile_t::PITCH;
  constexpr int after = BACK ? 0 : 1;
  __shared__ __attribute__((aligned(16))) T sB[2][kChunk * PITCH];
  const Work w = work_of(pl, pl.slots - 1);
  if (!w.live) return;
  const int64_t b = w.group / (int)p.heads;
  const int h = (int)(w.group - b * p.heads);
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, lr = lane & 15, pr = Mma<T>::row(lr);
  const int col = w.slice * kCols + wave * 16 + lr;
  const bool live = col < p.dc;
  const int64_t n = length_of(p, b);
  const int64_t lo = w.segment * pl.part_tokens;
  const int64_t end = lo + pl.part_tokens < n ? lo + pl.part_tokens : n;
  const int64_t first = BACK ? n - 1 - lo : lo, dir = BACK ? -1 : 1;
  const T* pb = p.b.p + b * p.b.b + (h / p.b.group) * p.b.h + first * p.b.t;
  const T* pc = p.c.p + b * p.c.b + (h / p.c.group) * p.c.h + first * p.c.t;
  const int ccol = live ? col : p.dc - 1;
  const int64_t tb = dir * p.b.t, tc = dir * p.c.t;
  acc_t S[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) S[kt] = (acc_t)((T)0);
  const T ld = p.log_decay[h];
  T wt[2][4];
  weights(wt, p.scale_b, ld, kChunk, after, g);
  T lam = power(ld, (int64_t)kChunk);
  tile_t k;
  T c[2][4], cn[2][4];
  k.prepare(tb, p.da);
  const int64_t total = end - lo;
  if (total > 0) {
    const int m = total < kChunk ? (int)total : kChunk;
    k.load(pb, tb, m, p.da);
    load_c<T, FAST>(cn, pc, tc, m, g, ccol, p.dc);
  }
  int turn = 0;
  for (int64_t at = 0; at < total; at += kChunk, turn ^= 1) {
    const int m = total - at < kChunk ? (int)(total - at) : kChunk;
    k.store(sB[turn], m, p.da);                             // (two buffers: one barrier a chunk)
    if (m < kChunk) { weights(wt, p.scale_b, ld, m, after, g); lam = power(ld, (int64_t)m); }
    take(c, cn, m, g);
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) c[jt][r] *= wt[jt][r];
    __syncthreads();
    if (at + kChunk < total) {
      const int64_t next = at + kChunk;
      const int mn = total - next < kChunk ? (int)(total - next) : kChunk;
      k.load(pb + next * tb, tb, mn, p.da);
      load_c<T, FAST>(cn, pc + next * tc, tc, mn, g, ccol, p.dc);
    }
    add_tokens<T, DA>(S, sB[turn], c, lam, pr, g);
  }
  if (!live) return;
  T* s1 = pl.states + ((int64_t)w.group * pl.slots + w.segment + 1) * p.da * p.dc + col;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * kt + 4 * g + r;
      if (d < p.da) s1[(int64_t)d * p.dc] = S[kt][r];
    }
}

// From the parts' shares to the states in front of the segments (the slots at multiples of `parts`): one lane per element of
// a head's state, BATCH slots on their way at a time (no load may pass the stores of the batch before).
template <typename T, int BATCH>
__device__ __forceinline__ void carry(T* at, int64_t per, int& k, T& s, T ld, int64_t n, const Plan<T>& pl) {
  for (; k + BATCH <= pl.slots; k += BATCH) {
    T v[BATCH];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) v[u] = at[(int64_t)(k + u) * per];
#pragma unroll
    for (int u = 0; u < BATCH; ++u) {
      int64_t len = n - (k + u - 1) * pl.part_tokens;
      len = len < 0 ? 0 : (len < pl.part_tokens ? len : pl.part_tokens);
      s = s * power(ld, len) + v[u];
      if ((k + u) % pl.parts == 0) at[(int64_t)(k + u) * per] = s;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void segment_states(Role<T> p, Plan<T> pl) {
  const int per = p.da * p.dc;
  const int blocks = (per + 255) / 256;
  const int group = (int)(blockIdx.x / (unsigned)blocks);
  const int i = (int)(blockIdx.x - (unsigned)group * (unsigned)blocks) * 256 + (int)threadIdx.x;
  if (i >= per) return;
  const int64_t b = group / (int)p.heads;
  const int h = (int)(group - b * p.heads);
  const int64_t n = length_of(p, b);
  const T ld = p.log_decay[h];
  const int r = i / p.dc, c = i - r * p.dc;
  T* at = pl.states + (int64_t)group * pl.slots * per + i;
  T s = p.s0 ? p.s0[b * p.s0_b + h * p.s0_h + r * p.s0_r + c * p.s0_c] : (T)0;
  at[0] = s;
  int k = 1;
  carry<T, 32>(at, per, k, s, ld, n, pl);
  carry<T, 8>(at, per, k, s, ld, n, pl);
  carry<T, 2>(at, per, k, s, ld, n, pl);
  carry<T, 1>(at, per, k, s, ld, n, pl);
}

static int workgroups_per_cu(const void* kernel) {
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, 256, 0) != hipSuccess || n < 1) { (void)hipGetLastError(); n = 1; }
  return n;
}

#ifndef MINSEG
#define MINSEG 2
#endif
template <typename T, int DA, bool BACK, bool FAST>
static int run_chunks(const Role<T>& p) {
  Plan<T> pl = {};
  pl.slices = (p.dc + kCols - 1) / kCols;
  pl.groups = (int)(p.batch * p.heads);
  pl.segments = 1;
  const int64_t wgs = (int64_t)pl.groups * pl.slices;
  const int64_t n_chunks = (p.tokens + kChunk - 1) / kChunk;
  // As many segments as the device has room for workgroups, of MINSEG chunks at least.
  static const int room = workgroups_per_cu((const void*)chunks<T, DA, BACK, FAST>), sums_room = workgroups_per_cu((const void*)segment_sums<T, DA, BACK, FAST>);
  int64_t segments = (int64_t)room * num_cus() / wgs;
  if (segments > n_chunks / MINSEG) segments = n_chunks / MINSEG;
  if (segments < 1) segments = 1;
  int64_t per_segment = n_chunks ? (n_chunks + segments - 1) / segments : 1;
  int64_t parts = 1;
  if (segments > 1) {
    // the sums run in parts of a segment, so that they too fill the device
    parts = (int64_t)sums_room * num_cus() / (wgs * (segments - 1));
    if (parts > per_segment / 2) parts = per_segment / 2;
    if (parts < 1) parts = 1;
    per_segment = (per_segment + parts - 1) / parts * parts;
  }
  pl.parts = (int)parts;
  pl.part_tokens = per_segment / parts * kChunk;
  pl.seg_tokens = per_segment * kChunk;
  pl.segments = (int)(n_chunks ? (n_chunks + per_segment - 1) / per_segment : 1);
  pl.slots = pl.parts * (pl.segments - 1) + 1;
  Scratch states;
  if (pl.segments > 1) {
    AM_TRY(states.take((size_t)pl.groups * pl.slots * p.da * p.dc * sizeof(T)));
    pl.states = (T*)states.p;
    const int64_t ids = ((int64_t)pl.groups * (pl.slots - 1) + 7) / 8 * 8 * pl.slices;
    hipLaunchKernelGGL((segment_sums<T, DA, BACK, FAST>), dim3((unsigned)ids), dim3(256), 0, stream(), p, pl);
    AM_TRY(check_launch("segment_sums"));
    hipLaunchKernelGGL((segment_states<T>), dim3((unsigned)(pl.groups * ((p.da * p.dc + 255) / 256))), dim3(256), 0, stream(), p, pl);
    AM_TRY(check_launch("segment_states"));
  }
  const int64_t ids = ((int64_t)pl.groups * pl.segments + 7) / 8 * 8 * pl.slices;
  hipLaunchKernelGGL((chunks<T, DA, BACK, FAST>), dim3((unsigned)ids), dim3(256), 0, stream(), p, pl);
  return check_launch("chunks");
}

template <typename T, int DA, bool BACK>
static int run_sized(const Role<T>& p) {
  // FAST: rows of whole vectors, and 32 tokens of every operand within 2^31 bytes
  const int64_t most = ((int64_t)1 << 31) / (kChunk * (int64_t)sizeof(T)) - kMostDim;
  auto near = [&](int64_t t) { return t < most && -t < most; };
  const bool fast = p.da % (16 / (int)sizeof(T)) == 0 && near(p.a.t) && near(p.b.t) && near(p.c.t) && near(p.o_t);
  return fast ? run_chunks<T, DA, BACK, true>(p) : run_chunks<T, DA, BACK, false>(p);
}

template <typename T, bool BACK>
static int run_role(const Role<T>& p) {
  if (p.da <= 32) return run_sized<T, 32, BACK>(p);
  if (p.da <= 64) return run_sized<T, 64, BACK>(p);
  if (p.da <= 96) return run_sized<T, 96, BACK>(p);
  if (p.da <= 128) return run_sized<T, 128, BACK>(p);
  if (p.da <= 192) return run_sized<T, 192, BACK>(p);
  return run_sized<T, 256, BACK>(p);
}

// One token: the state is read and written once. A workgroup takes one head's state in rows of 16-byte vectors: `lanes`
// lanes side by side on a row, 256 / lanes rows at once; the output is folded over the rows through LDS.
template <typename T> struct StepArgs {
  const T* q; int64_t q_b, q_h;
  const T* k; int64_t k_b, k_h;
  const T* v; int64_t v_b, v_h;
  T* state; int64_t s_b, s_h;
  T* out; int64_t o_b, o_h;
  const T* log_decay;
  T scale;
  int heads, group, dk, dv;
};

template <typename T, int V>
__global__ __launch_bounds__(256) void step(StepArgs<T> p, int lanes, int tiles) {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  __shared__ T fold[256 * V];
  const int64_t at = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x - at * tiles);
  const int64_t b = at / p.heads;
  const int h = (int)(at - b * p.heads);
  const int rows = 256 / lanes, row0 = (int)threadIdx.x / lanes;
  const int c = (tile * lanes + (int)threadIdx.x - row0 * lanes) * V;
  const bool live = row0 < rows && c < p.dv;
  const T* q = p.q + b * p.q_b + h * p.q_h;
  const T* k = p.k + b * p.k_b + (h / p.group) * p.k_h;
  const T lam = dev_exp(p.log_decay[h]);
  vec_t acc = (vec_t)((T)0);
  if (live) {
    const vec_t v = *(const vec_t*)(p.v + b * p.v_b + (h / p.group) * p.v_h + c);
    T* s = p.state + b * p.s_b + h * p.s_h + c;
#pragma unroll 4
    for (int r = row0; r < p.dk; r += rows) {
      vec_t w = *(vec_t*)(s + (int64_t)r * p.dv);
      w = w * lam + v * k[r];
      acc += w * q[r];
      *(vec_t*)(s + (int64_t)r * p.dv) = w;
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) fold[threadIdx.x * V + e] = acc[e];
  __syncthreads();
  if (!live || row0 != 0) return;
  T* out = p.out + b * p.o_b + h * p.o_h + c;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    T sum = acc[e];
    for (int r = 1; r < rows; ++r) sum += fold[(threadIdx.x + r * lanes) * V + e];
    out[e] = sum * p.scale;
  }
}

static int check_sizes(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv) {
  if (batch < 0 || tokens < 0 || heads < 0 || kv_heads < 0) return fail(AM_E_SHAPE, "%s: negative extent", fn);
  if (dk < 1 || dv < 1 || dk > kMostDim || dv > kMostDim)
    return fail(AM_E_SHAPE, "%s: heads of %lld and %lld elements (1 .. %lld are supported)", fn, (long long)dk, (long long)dv, (long long)kMostDim);
  if (heads && (kv_heads < 1 || heads % kv_heads)) return fail(AM_E_SHAPE, "%s: %lld heads cannot share %lld key / value heads evenly", fn, (long long)heads, (long long)kv_heads);
  if (heads && batch > ((int64_t)1 << 20) / heads) return fail(AM_E_SHAPE, "%s: more than 2^20 heads of all sequences together", fn);
  return AM_OK;
}

template <typename T> struct Strided { const T* p; int64_t b, t, h; };
template <typename T> struct Result { T* p; int64_t b, t, h; };
template <typename T> static bool broadcast_result(const Result<T>& r, int64_t batch, int64_t tokens, int64_t heads) {
  return tokens > 0 && ((batch > 1 && r.b == 0) || (tokens > 1 && r.t == 0) || (heads > 1 && r.h == 0));
}

template <typename T>
static int forward(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale,
                   const T* log_decay, const int64_t* lengths, Strided<T> q, Strided<T> k, Strided<T> v, const T* s0, int64_t s0_b,
                   int64_t s0_h, Result<T> out, T* s1, int64_t s1_b, int64_t s1_h) {
  AM_TRY(check_sizes(fn, batch, tokens, heads, kv_heads, dk, dv));
  if (batch == 0 || heads == 0) return AM_OK;
  if (!log_decay || (tokens && (!q.p || !k.p || !v.p || !out.p))) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if (broadcast_result(out, batch, tokens, heads) || (s1 && ((batch > 1 && s1_b == 0) || (heads > 1 && s1_h == 0))))
    return fail(AM_E_SHAPE, "%s: a result is a broadcast view", fn);
  AM_TRY(ensure_init());
  const int group = (int)(heads / kv_heads);
  Role<T> p = {};
  p.a = {q.p, q.b, q.t, q.h, 1};
  p.b = {k.p, k.b, k.t, k.h, group};
  p.c = {v.p, v.b, v.t, v.h, group};
  p.out = out.p; p.o_b = out.b; p.o_t = out.t; p.o_h = out.h;
  p.s0 = s0; p.s0_b = s0_b; p.s0_h = s0_h; p.s0_r = dv; p.s0_c = 1;
  p.s1 = s1; p.s1_b = s1_b; p.s1_h = s1_h; p.s1_r = dv; p.s1_c = 1;
  p.scale_a = scale; p.scale_b = (T)1;
  p.da = (int)dk; p.dc = (int)dv;
  p.log_decay = log_decay; p.lengths = lengths;
  p.batch = batch; p.tokens = tokens; p.heads = heads;
  return run_role<T, false>(p);
}

// out[b, t, head, :] = the sum of the `group` heads' shares that follow each other, in the heads' order
template <typename T, int V>
__global__ __launch_bounds__(256) void fold(const T* shares, Result<T> out, int64_t rows, int tokens, int kv_heads, int group, int d) {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  const int per = d / V;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = i / per;                             // (batch, token, head)
  if (row >= rows) return;
  const int c = (int)(i - row * per) * V;
  const T* q = shares + row * group * d + c;
  vec_t sum = *(const vec_t*)q;
  for (int m = 1; m < group; ++m) sum += *(const vec_t*)(q + (int64_t)m * d);
  const int64_t bt = row / kv_heads, b = bt / tokens;
  *(vec_t*)(out.p + b * out.b + (bt - b * tokens) * out.t + (row - bt * kv_heads) * out.h + c) = sum;
}

template <typename T>
static int fold_heads(const T* shares, const Result<T>& out, int64_t batch, int64_t tokens, int64_t kv_heads, int group, int d) {
  constexpr int W = 16 / (int)sizeof(T);
  const int64_t rows = batch * tokens * kv_heads;
  if (rows == 0) return AM_OK;
  const bool vec = d % W == 0 && (uintptr_t)out.p % 16 == 0 && out.b % W == 0 && out.t % W == 0 && out.h % W == 0;
  const int64_t wgs = (rows * (vec ? d / W : d) + 255) / 256;
  if (wgs >= ((int64_t)1 << 31) || tokens >= ((int64_t)1 << 31)) return fail(AM_E_SHAPE, "decay attention: too many tokens for shared heads");
  if (vec) hipLaunchKernelGGL((fold<T, W>), dim3((unsigned)wgs), dim3(256), 0, stream(), shares, out, rows, (int)tokens, (int)kv_heads, group, d);
  else hipLaunchKernelGGL((fold<T, 1>), dim3((unsigned)wgs), dim3(256), 0, stream(), shares, out, rows, (int)tokens, (int)kv_heads, group, d);
  return check_launch("fold");
}

template <typename T>
static int backward(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale,
                    const T* log_decay, const int64_t* lengths, Strided<T> go, Strided<T> q, Strided<T> k, Strided<T> v, const T* s0,
                    int64_t s0_b, int64_t s0_h, const T* gs, int64_t gs_b, int64_t gs_h, Result<T> dq, Result<T> dkey, Result<T> dval,
                    T* gs0, int64_t gs0_b, int64_t gs0_h) {
  AM_TRY(check_sizes(fn, batch, tokens, heads, kv_heads, dk, dv));
  if (batch == 0 || heads == 0) return AM_OK;
  if (!log_decay || (tokens && (!go.p || !q.p || !k.p || !v.p || !dq.p || !dkey.p || !dval.p))) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if (broadcast_result(dq, batch, tokens, heads) || broadcast_result(dkey, batch, tokens, kv_heads) || broadcast_result(dval, batch, tokens, kv_heads) ||
      (gs0 && ((batch > 1 && gs0_b == 0) || (heads > 1 && gs0_h == 0))))
    return fail(AM_E_SHAPE, "%s: a result is a broadcast view", fn);
  AM_TRY(ensure_init());
  const int group = (int)(heads / kv_heads);
  const Operand<T> Q = {q.p, q.b, q.t, q.h, 1}, G = {go.p, go.b, go.t, go.h, 1};
  const Operand<T> K = {k.p, k.b, k.t, k.h, group}, W = {v.p, v.b, v.t, v.h, group};
  Role<T> p = {};
  p.log_decay = log_decay; p.lengths = lengths;
  p.batch = batch; p.tokens = tokens; p.heads = heads;
  // dq: forwards over (do, v, k) from the transposed first state
  p.a = G; p.b = W; p.c = K;
  p.out = dq.p; p.o_b = dq.b; p.o_t = dq.t; p.o_h = dq.h;
  p.s0 = s0; p.s0_b = s0_b; p.s0_h = s0_h; p.s0_r = 1; p.s0_c = dv;
  p.scale_a = scale; p.scale_b = (T)1;
  p.da = (int)dv; p.dc = (int)dk;
  AM_TRY((run_role<T, false>(p)));
  // dk and dv: backwards. Where heads share a key / value head each writes its own share, and `fold_heads` adds them up.
  // dk first: dv's walk writes the first state's gradient, which may lie over the last state's.
  p.scale_a = (T)1; p.scale_b = scale;
  p.s0 = gs; p.s0_b = gs_b; p.s0_h = gs_h;
  Scratch shares;
  if (group > 1 && tokens) AM_TRY(shares.take((size_t)batch * tokens * heads * (dk > dv ? dk : dv) * sizeof(T)));
  auto into = [&](const Result<T>& r, int64_t d) {
    if (group == 1) { p.out = r.p; p.o_b = r.b; p.o_t = r.t; p.o_h = r.h; }
    else { p.out = (T*)shares.p; p.o_b = tokens * heads * d; p.o_t = heads * d; p.o_h = d; }
  };
  p.a = W; p.b = G; p.c = Q;
  into(dkey, dk);
  p.s0_r = 1; p.s0_c = dv;
  p.da = (int)dv; p.dc = (int)dk;
  AM_TRY((run_role<T, true>(p)));
  if (group > 1) AM_TRY(fold_heads((const T*)shares.p, dkey, batch, tokens, kv_heads, group, (int)dk));
  p.a = K; p.b = Q; p.c = G;
  into(dval, dv);
  p.s0_r = dv; p.s0_c = 1;
  p.s1 = gs0; p.s1_b = gs0_b; p.s1_h = gs0_h; p.s1_r = dv; p.s1_c = 1;
  p.da = (int)dk; p.dc = (int)dv;
  AM_TRY((run_role<T, true>(p)));
  if (group > 1) AM_TRY(fold_heads((const T*)shares.p, dval, batch, tokens, kv_heads, group, (int)dv));
  return AM_OK;
}

template <typename T>
static int one_step(const char* fn, int64_t batch, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale, const T* log_decay,
                    const T* q, int64_t q_b, int64_t q_h, const T* k, int64_t k_b, int64_t k_h, const T* v, int64_t v_b, int64_t v_h,
                    T* state, int64_t s_b, int64_t s_h, T* out, int64_t o_b, int64_t o_h) {
  AM_TRY(check_sizes(fn, batch, 1, heads, kv_heads, dk, dv));
  if (batch == 0 || heads == 0) return AM_OK;
  if (!log_decay || !q || !k || !v || !state || !out) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if ((batch > 1 && (s_b == 0 || o_b == 0)) || (heads > 1 && (s_h == 0 || o_h == 0))) return fail(AM_E_SHAPE, "%s: the state or the result is a broadcast view", fn);
  AM_TRY(ensure_init());
  StepArgs<T> p = {q, q_b, q_h, k, k_b, k_h, v, v_b, v_h, state, s_b, s_h, out, o_b, o_h, log_decay, scale, (int)heads, (int)(heads / kv_heads), (int)dk, (int)dv};
  constexpr int W = 16 / (int)sizeof(T);
  auto fits = [&](const void* base, int64_t sb, int64_t sh) {
    return (uintptr_t)base % 16 == 0 && (sb % W == 0 || batch == 1) && (sh % W == 0 || heads == 1);
  };
  const bool vec = dv % W == 0 && fits(v, v_b, v_h) && fits(state, s_b, s_h);
  const int units = vec ? (int)dv / W : (int)dv;
  // narrower columns where the heads alone would leave CUs without work
  int lanes = units < 64 ? units : 64;
  while (lanes > 8 && batch * heads * ((units + lanes - 1) / lanes) < 2 * num_cus()) lanes = (lanes + 1) / 2;
  const int tiles = (units + lanes - 1) / lanes;
  const int64_t wgs = batch * heads * tiles;
  if (wgs >= ((int64_t)1 << 31)) return fail(AM_E_SHAPE, "%s: too many heads for one launch", fn);
  if (vec) hipLaunchKernelGGL((step<T, W>), dim3((unsigned)wgs), dim3(256), 0, stream(), p, lanes, tiles);
  else hipLaunchKernelGGL((step<T, 1>), dim3((unsigned)wgs), dim3(256), 0, stream(), p, lanes, tiles);
  return check_launch("step");
}

}  // namespace decay
}  // namespace am

using namespace am;

#define AM_DECAY_ATTENTION(S, T)                                                                                                      \
  extern "C" int am_hip_decay_attention_##S(                                                                                          \
      int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale, const T* log_decay,            \
      const int64_t* lengths, const T* q, int64_t q_b, int64_t q_t, int64_t q_h, const T* k, int64_t k_b, int64_t k_t, int64_t k_h,   \
      const T* v, int64_t v_b, int64_t v_t, int64_t v_h, const T* state_in, int64_t si_b, int64_t si_h, T* out, int64_t o_b,          \
      int64_t o_t, int64_t o_h, T* state_out, int64_t so_b, int64_t so_h) {                                                           \
    return decay::forward<T>("am_hip_decay_attention_" #S, batch, tokens, heads, kv_heads, dk, dv, scale, log_decay, lengths,         \
                             {q, q_b, q_t, q_h}, {k, k_b, k_t, k_h}, {v, v_b, v_t, v_h}, state_in, si_b, si_h, {out, o_b, o_t, o_h}, \
                             state_out, so_b, so_h);                                                                                  \
  }                                                                                                                                   \
  extern "C" int am_hip_decay_attention_backward_##S(                                                                                 \
      int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale, const T* log_decay,            \
      const int64_t* lengths, const T* grad_out, int64_t g_b, int64_t g_t, int64_t g_h, const T* q, int64_t q_b, int64_t q_t,         \
      int64_t q_h, const T* k, int64_t k_b, int64_t k_t, int64_t k_h, const T* v, int64_t v_b, int64_t v_t, int64_t v_h,              \
      const T* state_in, int64_t si_b, int64_t si_h, const T* grad_state_out, int64_t gso_b, int64_t gso_h, T* grad_q, int64_t gq_b,  \
      int64_t gq_t, int64_t gq_h, T* grad_k, int64_t gk_b, int64_t gk_t, int64_t gk_h, T* grad_v, int64_t gv_b, int64_t gv_t,         \
      int64_t gv_h, T* grad_state_in, int64_t gsi_b, int64_t gsi_h) {                                                                 \
    return decay::backward<T>("am_hip_decay_attention_backward_" #S, batch, tokens, heads, kv_heads, dk, dv, scale, log_decay,        \
                              lengths, {grad_out, g_b, g_t, g_h}, {q, q_b, q_t, q_h}, {k, k_b, k_t, k_h}, {v, v_b, v_t, v_h},         \
                              state_in, si_b, si_h, grad_state_out, gso_b, gso_h, {grad_q, gq_b, gq_t, gq_h},                         \
                              {grad_k, gk_b, gk_t, gk_h}, {grad_v, gv_b, gv_t, gv_h}, grad_state_in, gsi_b, gsi_h);                   \
  }                                                                                                                                   \
  extern "C" int am_hip_decay_attention_step_##S(                                                                                     \
      int64_t batch, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale, const T* log_decay, const T* q, int64_t q_b,   \
      int64_t q_h, const T* k, int64_t k_b, int64_t k_h, const T* v, int64_t v_b, int64_t v_h, T* state, int64_t s_b, int64_t s_h,    \
      T* out, int64_t o_b, int64_t o_h) {                                                                                             \
    return decay::one_step<T>("am_hip_decay_attention_step_" #S, batch, heads, kv_heads, dk, dv, scale, log_decay, q, q_b, q_h, k,    \
                              k_b, k_h, v, v_b, v_h, state, s_b, s_h, out, o_b, o_h);                                                 \
  }

AM_DECAY_ATTENTION(f32, float)
AM_DECAY_ATTENTION(f64, double)
