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

// e^{g n} for a state that is multiplied by it chunk after chunk. Its rounding would be the same every time and add up over the walk:
// with g = -10^-6 a float e^{32 g} is off by up to 2^-25, and after 1024 chunks the state by 3 * 10^-5. So the exponential is made in
// double and kept with what its rounding lost, and every chunk takes the float next to it that pays off the debt of those before: the
// product over any stretch of chunks is right to a float's step. (In the state's own product, as a sum of two floats, the same costs
// every element an instruction or two: prompts of 4 x 4096 tokens, 16 heads of 128 x 128, 220.8 -> 228.3 us.)
struct Rounded { float hi, lo; };
__device__ __forceinline__ Rounded rounded(double e) { const float hi = (float)e; return {hi, (float)(e - (double)hi)}; }
__device__ __forceinline__ float next_factor(Rounded f, float& debt) {
  debt += f.lo;
  const float lam = f.hi + debt;
  debt -= lam - f.hi;
  return lam;
}

// ---- chunks of 32 tokens on the matrix cores ---------------------------------------------------------------------------
//
// For the tokens of a chunk, i and j counted within it, and the state S in front of it,
//     o_i = sum_{j <= i} A_ij c_j + e^{g (i + after)} a_i S      A_ij = e^{g (i - j)} (a_i . b_j)
//     S <- e^{g N} S + sum_j e^{g (N - after - j)} b_j^T c_j
// so a chunk is four products: a b^T (32 x 32), A c, a S and b^T c. A workgroup walks the chunks of one head, a wavefront
// owning columns of S and of o for all da rows (or half of them, below), as accumulators in its registers: the product
// instructions leave neighbouring rows of a result in a lane, and the sum over k may take its k in any order that both
// operands share, so the rows of S a lane holds are k of the next product's right operand as they stand.
// Registers run out, and a few to some hundred of them are spilled, where rows are no whole vectors of 16 bytes (an address of 64
// bits for every element) and in float64 from 192 rows on; tests/test_sequence_resources.py holds the list. us of prompt +
// gradients, 4 x 4096 tokens, 16 heads in float32: of 128 x 128 218 + 591, of 126 x 126 376 + 1049; 2 x 1024 tokens, 8 heads in
// float64: of 128 x 128 68 + 170, of 192 x 192 154 + 416, of 256 x 256 240 + 623.
//   - a b^T is computed transposed, so that a lane's four values lie next to each other in a row of A in LDS; the three
//     tiles on and under the diagonal go to three wavefronts.
//   - c is read straight into the layout of a right operand, which A c and b^T c share.
// a and b go through LDS; the next chunk's are on their way in registers meanwhile. All exponents of e^g are differences that
// the mask leaves >= 0, so nothing overflows however long the text.
//
// float64 runs on the 16 x 16 x 4 product of doubles (`chunks_f64`). float32 does not run on its float counterpart, which has
// a sixteenth of the bfloat16 rate: every operand is the sum of three bfloat16 (8 bits each, 24 in all: `split`), and a
// product takes the six pairs of pieces down to 2^-16 (the three that are left out are below 2^-24 of the term, a float's
// half step), with float32 sums inside the instruction: `chunks_f32`. Measured on 4 x 4096 tokens, 16 heads of 128 x 128:
// 291 us with the float instruction, 223 us in pieces, both before the steps noted at the kernels below; with them 212.
//
// Where the heads alone do not fill the device, the tokens are cut into segments: `sums_*` add up each segment's share of the
// state, `segment_states` carries them from segment to segment, and the chunk kernels start every segment from its own.
constexpr int64_t kMostDim = 256;
constexpr int kChunk = 32;
constexpr int kLds = 160 * 1024;

template <typename T> struct Plan {
  T* states;                   // [batch * heads][slots][da * dc]: the state in front of each part; null: one segment
  int st_r, st_c;              // strides of a state's rows and columns there
  int segments, slices;
  int parts, slots;            // parts of a segment; slots = parts * (segments - 1) + 1, one in front of every part but the last segment's later ones
  int64_t seg_tokens, part_tokens;   // multiples of kChunk, seg_tokens = parts * part_tokens
  int groups;                  // batch * heads
};

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

// The stretch of a head's walk that a workgroup takes: local tokens lo .. lo + total, local token i being token i or, walking
// back, n - 1 - i. The pointers are those of the first one, t_* the steps to the next.
template <typename T, bool BACK> struct Path {
  int64_t b, n, lo, hi, total;
  int h;
  const T *a, *k, *c;
  T* o;
  int64_t ta, tk, tc, to;
  __device__ __forceinline__ Path(const Role<T>& p, int group, int64_t lo_, int64_t tokens) {
    b = group / (int)p.heads;
    h = (int)(group - b * p.heads);
    n = length_of(p, b);
    lo = lo_;
    hi = lo + tokens < p.tokens ? lo + tokens : p.tokens;
    total = (hi < n ? hi : n) - lo;
    const int64_t first = BACK ? n - 1 - lo : lo, dir = BACK ? -1 : 1;
    a = p.a.p + b * p.a.b + (h / p.a.group) * p.a.h + first * p.a.t;
    k = p.b.p + b * p.b.b + (h / p.b.group) * p.b.h + first * p.b.t;
    c = p.c.p + b * p.c.b + (h / p.c.group) * p.c.h + first * p.c.t;
    o = p.out + b * p.o_b + h * p.o_h + first * p.o_t;
    ta = dir * p.a.t; tk = dir * p.b.t; tc = dir * p.c.t; to = dir * p.o_t;
  }
  // tokens of the chunk at local token `at`, 1 .. 32
  __device__ __forceinline__ int tokens(int64_t at) const { return total - at < kChunk ? (int)(total - at) : kChunk; }
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
template <typename T, int DA, bool FAST, int THREADS> struct Tile {
  static constexpr int V = 16 / (int)sizeof(T), PER_ROW = DA / V, ALL = kChunk * PER_ROW, NV = (ALL + THREADS - 1) / THREADS;
  static constexpr bool EVEN = THREADS % PER_ROW == 0;   // vector u of a lane lies whole rows behind its first
  static constexpr bool FULL = ALL % THREADS == 0;       // every lane has NV vectors (else the last ones repeat the tile's last)
  static constexpr int NO = EVEN && FULL ? 1 : NV;
  typedef T vec_t __attribute__((ext_vector_type(V)));
  vec_t v[NV];
  uint32_t off[NO];                                      // of a lane's vectors behind the chunk's first token

  static __device__ __forceinline__ int vector(int u) {
    const int f = (int)threadIdx.x + u * THREADS;
    return FULL || f < ALL ? f : ALL - 1;
  }
  __device__ __forceinline__ void prepare(int64_t step) {
    if constexpr (FAST) {
#pragma unroll
      for (int u = 0; u < NO; ++u) {
        const int f = vector(u), row = f / PER_ROW, c = (f - row * PER_ROW) * V;
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
        const uint32_t o = NO == 1 ? off[0] + (k.first + (uint32_t)(u * (THREADS / PER_ROW) * (int)step * (int)sizeof(T))) : off[u % NO] + k.first;
        v[u] = __builtin_bit_cast(vec_t, __builtin_amdgcn_raw_buffer_load_b128(k.rsrc, (int)o, 0, 0));
      }
    } else {
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        const int f = vector(u);
        int row = f / PER_ROW, c = (f - row * PER_ROW) * V;
        row = row < n ? row : n - 1;
        const T* q = p + row * step;
#pragma unroll
        for (int e = 0; e < V; ++e) v[u][e] = q[c + e < da ? c + e : da - 1];
      }
    }
  }
  // write(row, column, vector) for every vector of the lane
  template <typename F> __device__ __forceinline__ void store(int n, int da, F write) const {
    const bool all = n == kChunk && da == DA;
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int f = vector(u), row = f / PER_ROW, c = (f - row * PER_ROW) * V;
      vec_t w = v[u];
      if (!all) {
#pragma unroll
        for (int e = 0; e < V; ++e) w[e] = (row < n && c + (FAST ? 0 : e) < da) ? w[e] : (T)0;
      }
      write(row, c, w);
    }
  }
};

// Nothing moves across here: the LDS reads of the next step stay in front of the matrix instructions of this one. Left alone,
// the scheduler puts every read right in front of its use, and the wavefront waits for LDS in every step.
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// v, computed where it stands: what depends on it is not kept in registers over the loop around it.
__device__ __forceinline__ uint32_t here(uint32_t v) { asm volatile("" : "+v"(v)); return v; }

// c of a chunk of n >= 1 tokens, in the layout of a right operand: register r of tile jt is token 16 jt + 4 g + r, in column
// `col`. `take` makes tokens behind the n-th 0.
template <typename T, bool FAST>
__device__ __forceinline__ void load_c(T (&c)[2][4], const T* p, int64_t step, int n, int g, int col, int width) {
  if constexpr (FAST) {
    const Chunk k = chunk_of(p, step, n, width);
    const uint32_t off = here((uint32_t)((4 * g * (int)step + col) * (int)sizeof(T)));
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

// The lane's column of a chunk's result: register r of tile it is token 16 it + 4 g + r.
template <typename T, typename A, bool FAST, int TILES>
__device__ __forceinline__ void put_o(const A (&o)[TILES], T* p, int64_t step, int n, int g, int col, int width) {
  if constexpr (FAST) {
    const Chunk k = chunk_of(p, step, n, width);
    const uint32_t off = here((uint32_t)((4 * g * (int)step + col) * (int)sizeof(T)));
#pragma unroll
    for (int it = 0; it < TILES; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) put(k, off + (k.first + (uint32_t)((16 * it + r) * (int)step * (int)sizeof(T))), o[it][r]);
  } else {
#pragma unroll
    for (int it = 0; it < TILES; ++it)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * it + 4 * g + r;
        if (i < n) p[i * step + col] = o[it][r];
      }
  }
}

// Zeros into the lane's column behind the sequence, as far as the stretch goes.
template <typename T, bool BACK>
__device__ __forceinline__ void zero_tail(const Role<T>& p, const Path<T, BACK>& path, int g, int col) {
  T* o = p.out + path.b * p.o_b + path.h * p.o_h + col;
  for (int64_t t = (path.lo > path.n ? path.lo : path.n) + g; t < path.hi; t += 4) o[t * p.o_t] = (T)0;
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

// The factors of a lane's rows: reach, e^{g (i + after)} of its rows of o; mask, e^{g (i - j)} or 0 of its row j, column i of a
// transposed tile of A at distance 0 and 1; both with the scales in.
template <typename T>
__device__ __forceinline__ void row_factors(T (&reach)[2][4], T (&mask)[2][4], const Role<T>& p, T ld, int after, int g, int lr) {
#pragma unroll
  for (int it = 0; it < 2; ++it)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      reach[it][r] = p.scale_a * power(ld, (int64_t)(16 * it + 4 * g + r + after));
      const int apart = 16 * it + lr - 4 * g - r;
      mask[it][r] = apart >= 0 ? p.scale_a * p.scale_b * power(ld, (int64_t)apart) : (T)0;
    }
}

// Where the first state of a segment is read, and its strides.
template <typename T> struct First { const T* p; int64_t r, c; };
template <typename T> __device__ __forceinline__ First<T> first_state(const Role<T>& p, const Plan<T>& pl, const Work& w, int64_t b, int h) {
  if (pl.states) return {pl.states + ((int64_t)w.group * pl.slots + w.segment * pl.parts) * p.da * p.dc, pl.st_r, pl.st_c};
  return {p.s0 ? p.s0 + b * p.s0_b + h * p.s0_h : nullptr, p.s0_r, p.s0_c};
}

// ---- float64 ----
// A lane's four registers of a 16 x 16 result are rows 4 i + g there (i the register, g = lane / 16). The rows that lanes bring
// as left operand are ordered so that they are rows 4 g + i all the same, and a left operand's four k lie side by side in LDS.
typedef double acc64 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ acc64 mma64(double a, double b, acc64 c) { return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0); }
__device__ __forceinline__ int row64(int r) { return 4 * (r & 3) + (r >> 2); }
constexpr int kWaves64 = 4, kCols64 = 16 * kWaves64;    // wavefronts and columns of a workgroup

__device__ __forceinline__ void four(const double* lds, double (&out)[4]) {
  typedef double d2 __attribute__((ext_vector_type(2)));
  const d2 a = *(const d2*)lds, b = *(const d2*)(lds + 2);
  out[0] = a[0]; out[1] = a[1]; out[2] = b[0]; out[3] = b[1];
}

// One wavefront's share of a chunk's sum over the tokens: S <- e^{g N} S + b^T (w c), c given weighted.
template <int DA>
__device__ __forceinline__ void add_tokens64(acc64 (&S)[DA / 16], const double* sB, const double (&wc)[2][4], double lam, int pr, int g) {
  constexpr int PITCH = DA + 2;
#pragma unroll
  for (int kt = 0; kt < DA / 16; ++kt) {
    S[kt] *= lam;
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        S[kt] = mma64(sB[(16 * jt + 4 * g + r) * PITCH + 16 * kt + pr], wc[jt][r], S[kt]);
  }
}

template <int DA, bool BACK, bool FAST>
__global__ __launch_bounds__(256, DA <= 64 ? 2 : 1) void chunks_f64(Role<double> p, Plan<double> pl) {
  constexpr int KT = DA / 16, PITCH = DA + 2, APITCH = kChunk + 2;
  constexpr int after = BACK ? 0 : 1;
  constexpr int BUFS = (4 * kChunk * PITCH + kChunk * APITCH) * 8 <= kLds ? 2 : 1;
  __shared__ __attribute__((aligned(16))) double bufs[BUFS][2][kChunk * PITCH];
  __shared__ __attribute__((aligned(16))) double sA[kChunk * APITCH];
  const Work w = work_of(pl, pl.segments);
  if (!w.live) return;
  const Path<double, BACK> path(p, w.group, w.segment * pl.seg_tokens, pl.seg_tokens);
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, lr = lane & 15, pr = row64(lr);
  const int col = w.slice * kCols64 + wave * 16 + lr;
  const bool live = col < p.dc;
  const int ccol = live ? col : p.dc - 1;
  acc64 S[KT];
  const First<double> s0 = first_state(p, pl, w, path.b, path.h);
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * kt + 4 * g + r;
      S[kt][r] = (s0.p && live && d < p.da) ? s0.p[d * s0.r + col * s0.c] : 0.0;
    }
  const double ld = p.log_decay[path.h];
  double reach[2][4], mask[2][4], wt[2][4];
  row_factors(reach, mask, p, ld, after, g, lr);
  weights(wt, p.scale_b, ld, kChunk, after, g);
  double lam = power(ld, (int64_t)kChunk);

  Tile<double, DA, FAST, 256> a, k;
  double c[2][4], cn[2][4];
  a.prepare(path.ta);
  k.prepare(path.tk);
  auto fetch = [&](int64_t at) {
    const int m = path.tokens(at);
    a.load(path.a + at * path.ta, path.ta, m, p.da);
    k.load(path.k + at * path.tk, path.tk, m, p.da);
    load_c<double, FAST>(cn, path.c + at * path.tc, path.tc, m, g, ccol, p.dc);
  };
  auto stage = [&](double (&to)[2][kChunk * PITCH], int m) {
    typedef double d2 __attribute__((ext_vector_type(2)));
    a.store(m, p.da, [&](int row, int cc, d2 v) { *(d2*)(to[0] + row * PITCH + cc) = v; });
    k.store(m, p.da, [&](int row, int cc, d2 v) { *(d2*)(to[1] + row * PITCH + cc) = v; });
  };
  if (path.total > 0) { fetch(0); stage(bufs[0], path.tokens(0)); }
  int turn = 0;
  for (int64_t at = 0; at < path.total; at += kChunk) {
    const int64_t next = at + kChunk;
    const int m = path.tokens(at);
    const double* sQ = bufs[turn][0];
    const double* sB = bufs[turn][1];
    take(c, cn, m, g);
    __syncthreads();
    if (next < path.total) fetch(next);
    if (wave < 3) {                                         // tiles (0, 0), (1, 0), (1, 1) of A
      const int it = wave ? 1 : 0, jt = wave == 2 ? 1 : 0;
      acc64 t = (acc64)(0.0);
      const double* px = sB + (16 * jt + pr) * PITCH + 4 * g;
      const double* py = sQ + (16 * it + lr) * PITCH + 4 * g;
      double x[2][4], y[2][4];
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
        for (int r = 0; r < 4; ++r) t = mma64(x[kt & 1][r], y[kt & 1][r], t);
        pin();
      }
      double* q = sA + (16 * it + lr) * APITCH + 16 * jt + 4 * g;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool under = it > jt || lr >= 4 * g + r;      // a choice, not a product with 0: the term above may be a NaN
        q[r] = under ? t[r] * (it > jt ? mask[1][r] : mask[0][r]) : 0.0;
      }
    }
    acc64 o[2];
    {
      const double* px = sQ + pr * PITCH + 4 * g;
      double x[2][2][4];
      o[0] = o[1] = (acc64)(0.0);
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
          o[0] = mma64(x[kt & 1][0][r], S[kt][r], o[0]);
          o[1] = mma64(x[kt & 1][1][r], S[kt][r], o[1]);
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
      const double* px = sA + pr * APITCH + 4 * g;
      double x[3][4];
      four(px, x[0]);
      four(px + 16 * APITCH, x[1]);
      four(px + 16 * APITCH + 16, x[2]);
      pin();
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        o[0] = mma64(x[0][r], c[0][r], o[0]);
        o[1] = mma64(x[1][r], c[0][r], o[1]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) o[1] = mma64(x[2][r], c[1][r], o[1]);
    }
    if (m < kChunk) { weights(wt, p.scale_b, ld, m, after, g); lam = power(ld, (int64_t)m); }
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) c[jt][r] *= wt[jt][r];
    add_tokens64<DA>(S, sB, c, lam, pr, g);
    if (live) put_o<double, acc64, FAST, 2>(o, path.o + at * path.to, path.to, m, g, col, p.dc);
    // the next chunk into LDS: into the other buffer, or (where two do not fit) behind a barrier
    if constexpr (BUFS == 2) turn ^= 1;
    else __syncthreads();
    if (next < path.total) stage(bufs[turn], path.tokens(next));
  }
  if (live) zero_tail(p, path, g, col);
  if (p.s1 && w.segment == pl.segments - 1 && live) {
    double* s1 = p.s1 + path.b * p.s1_b + path.h * p.s1_h + col * p.s1_c;
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
template <int DA, bool BACK, bool FAST>
__global__ __launch_bounds__(256) void sums_f64(Role<double> p, Plan<double> pl) {
  constexpr int KT = DA / 16, PITCH = DA + 2;
  constexpr int after = BACK ? 0 : 1;
  __shared__ __attribute__((aligned(16))) double sB[2][kChunk * PITCH];
  const Work w = work_of(pl, pl.slots - 1);
  if (!w.live) return;
  const Path<double, BACK> path(p, w.group, w.segment * pl.part_tokens, pl.part_tokens);
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, lr = lane & 15, pr = row64(lr);
  const int col = w.slice * kCols64 + wave * 16 + lr;
  const bool live = col < p.dc;
  const int ccol = live ? col : p.dc - 1;
  acc64 S[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) S[kt] = (acc64)(0.0);
  const double ld = p.log_decay[path.h];
  double wt[2][4];
  weights(wt, p.scale_b, ld, kChunk, after, g);
  double lam = power(ld, (int64_t)kChunk);
  Tile<double, DA, FAST, 256> k;
  double c[2][4], cn[2][4];
  k.prepare(path.tk);
  auto fetch = [&](int64_t at) {
    const int m = path.tokens(at);
    k.load(path.k + at * path.tk, path.tk, m, p.da);
    load_c<double, FAST>(cn, path.c + at * path.tc, path.tc, m, g, ccol, p.dc);
  };
  if (path.total > 0) fetch(0);
  int turn = 0;
  for (int64_t at = 0; at < path.total; at += kChunk, turn ^= 1) {
    typedef double d2 __attribute__((ext_vector_type(2)));
    const int m = path.tokens(at);
    double* to = sB[turn];                                  // (two buffers: one barrier a chunk)
    k.store(m, p.da, [&](int row, int cc, d2 v) { *(d2*)(to + row * PITCH + cc) = v; });
    if (m < kChunk) { weights(wt, p.scale_b, ld, m, after, g); lam = power(ld, (int64_t)m); }
    take(c, cn, m, g);
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) c[jt][r] *= wt[jt][r];
    __syncthreads();
    if (at + kChunk < path.total) fetch(at + kChunk);
    add_tokens64<DA>(S, sB[turn], c, lam, pr, g);
  }
  if (!live) return;
  double* s1 = pl.states + ((int64_t)w.group * pl.slots + w.segment + 1) * p.da * p.dc + col;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 16 * kt + 4 * g + r;
      if (d < p.da) s1[(int64_t)d * p.dc] = S[kt][r];
    }
}

// ---- float32 ----
// The 16 x 16 x 32 product of bfloat16: a lane brings eight k of row (column) lane % 16 and gets rows 4 g + i of the result,
// g = lane / 16. Its k may be any eight as long as both operands agree:
//   - over da: k = 32 m + 8 g + e. The rows of S's tiles are ordered to match: registers i of tiles 2 m and 2 m + 1 are rows
//     32 m + 8 g + i and 32 m + 8 g + 4 + i, the eight that the lane needs when S is the right operand.
//   - over the chunk's tokens: the four j = 4 g + e, then the four 16 + 4 g + e, which is how c is loaded and how a lane holds
//     a transposed tile pair of A. b^T wants four tokens of one column there: the transposing LDS read gathers them from the
//     row-major pieces of b (lane i of sixteen points at row i / 4, four columns i % 4; it gets column i of the 4 x 16 block).
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef float acc32 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// x = out[0] + out[1] + out[2] up to 2^-27 |x|, each rounded to nearest: the residues are exact. (A residue below the smallest
// normal bfloat16 is lost: elements below 2^-108 keep 16 bits or fewer.)
template <typename V, int N> __device__ __forceinline__ void split(const float (&x)[N], V (&out)[3]) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    f32x2 v = {x[i], x[i + 1]};
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      const bf2 t = __builtin_convertvector(v, bf2);
      out[q][i] = t[0];
      out[q][i + 1] = t[1];
      v -= __builtin_convertvector(t, f32x2);
    }
  }
}

// c + x y, the six pairs of pieces that count, small ones first
__device__ __forceinline__ acc32 mma6(const bf8 (&x)[3], const bf8 (&y)[3], acc32 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[2], y[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], y[2], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], y[1], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[1], y[0], c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], y[1], c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x[0], y[0], c, 0, 0, 0);
}

// Pieces of 32 rows in LDS, rows padded by 32 bytes (against 16 the transposing reads conflict more: 238 -> 227 us for the
// gradients of 4 x 2048 tokens, 16 heads of 64 x 128).
template <int DA> struct Pieces {
  static constexpr int PITCH = DA + 16;
  __bf16 at[3][kChunk * PITCH];
  template <typename TILE> __device__ __forceinline__ void fill(const TILE& t, int n, int da) {
    t.store(n, da, [&](int row, int c, f32x4 v) {
      const float x[4] = {v[0], v[1], v[2], v[3]};
      bf4 q[3];
      split(x, q);
#pragma unroll
      for (int i = 0; i < 3; ++i) *(bf4*)(at[i] + row * PITCH + c) = q[i];
    });
  }
  // eight neighbouring elements
  __device__ __forceinline__ void row8(int row, int c, bf8 (&x)[3]) const {
#pragma unroll
    for (int i = 0; i < 3; ++i) x[i] = *(const bf8*)(at[i] + row * PITCH + c);
  }
  // left operand of b^T's rows 32 m + 4 t + 8 (lr / 4) + lr % 4 over the chunk's tokens
  __device__ __forceinline__ void tokens8(int m, int t, int g, int lr, bf8 (&x)[3]) const {
    typedef short s4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s4 lds4;
    const int where = (4 * g + (lr >> 2)) * PITCH + 32 * m + 8 * (lr & 3) + 4 * t;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const bf4 lo = __builtin_bit_cast(bf4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at[i] + where)));
      const bf4 hi = __builtin_bit_cast(bf4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(at[i] + where + 16 * PITCH)));
      x[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
};

// S <- e^{g N} S + b^T (w c) of a wavefront's 16 columns and its rows from 32 m on, c given weighted.
template <int DA, int KT>
__device__ __forceinline__ void add_tokens32(acc32 (&S)[KT], const Pieces<DA>& sB, const float (&wc)[2][4], float lam, int m, int g, int lr) {
  const float v[8] = {wc[0][0], wc[0][1], wc[0][2], wc[0][3], wc[1][0], wc[1][1], wc[1][2], wc[1][3]};
  bf8 y[3];
  split(v, y);
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) {
    bf8 x[3];
    sB.tokens8(m + (kt >> 1), kt & 1, g, lr, x);
    S[kt] = mma6(x, y, S[kt] * lam);
  }
}

// Wavefronts of a workgroup: eight for 128 columns; four for 64, or eight that halve the rows of the state (HALVES): two of them
// share columns, each adds up a S over its rows and finishes one of the two tiles of o. A chunk is a chain (LDS, split, product,
// barrier) that one wavefront spends mostly waiting in, so the registers are held down to let four share a SIMD wherever LDS has
// room for their workgroups. 4 x 4096 tokens, 16 heads of 128 x 128: 145 us of 112 that q, k, v and o take at a copy's rate,
// 2.1 GHz, vector instructions 58 % and matrix instructions 40 % of the cycles, LDS about as much; with two tiles of columns a
// wavefront, and half the wavefronts, 168 us; with the residues of `split` as two-element dot products (seven instructions for
// two elements in place of eleven) the same 145.
template <int DA, int WAVES> constexpr int kWaves = WAVES == 8 ? (DA <= 128 ? 4 : 2) : (DA <= 32 ? 4 : DA <= 64 ? 3 : 2);

template <int DA, int WAVES, int HALVES, bool BACK, bool FAST>
__global__ __launch_bounds__(64 * WAVES, (kWaves<DA, WAVES>)) void chunks_f32(Role<float> p, Plan<float> pl) {
  constexpr int KT = DA / 16 / HALVES, CT = WAVES / HALVES, APITCH = kChunk + 8;
  constexpr int after = BACK ? 0 : 1;
  __shared__ __attribute__((aligned(16))) Pieces<DA> sQ, sB;
  __shared__ __attribute__((aligned(16))) __bf16 sA[3][kChunk * APITCH];
  __shared__ __attribute__((aligned(16))) acc32 sX[HALVES == 2 ? WAVES : 1][64];
  __shared__ float sP[kChunk + 1];                          // e^{g n}: read when wanted, for the registers' sake
  __shared__ Rounded sF;                                    // e^{32 g}
  const Work w = work_of(pl, pl.segments);
  if (!w.live) return;
  const Path<float, BACK> path(p, w.group, w.segment * pl.seg_tokens, pl.seg_tokens);
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
  const int half = HALVES == 2 ? wave / CT : 0, m0 = half * (KT / 2);
  const int col = (w.slice * CT + wave % CT) * 16 + lr;
  const bool live = col < p.dc;
  const int ccol = live ? col : p.dc - 1;
  acc32 S[KT];
  const First<float> s0 = first_state(p, pl, w, path.b, path.h);
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 32 * (m0 + (kt >> 1)) + 8 * g + 4 * (kt & 1) + r;
      S[kt][r] = (s0.p && live && d < p.da) ? s0.p[d * s0.r + col * s0.c] : 0.0f;
    }
  const float ld = p.log_decay[path.h];
  const int at_it = wave ? 1 : 0, at_jt = wave == 2 ? 1 : 0;  // the first three wavefronts' tiles of A: (0, 0), (1, 0), (1, 1)
  if ((int)threadIdx.x <= kChunk) sP[threadIdx.x] = power(ld, (int64_t)threadIdx.x);
  if (threadIdx.x == 0) sF = rounded(power((double)ld, (int64_t)kChunk));
  float debt = 0.0f;
  const float ab = p.scale_a * p.scale_b;
  // A's rows 0 .. 15 have no tokens 16 .. 31: zeros once
  for (int i = (int)threadIdx.x; i < 3 * 16 * APITCH; i += 64 * WAVES) sA[i / (16 * APITCH)][i % (16 * APITCH)] = (__bf16)0.0f;

  Tile<float, DA, FAST, 64 * WAVES> a, k;
  float c[2][4];
  a.prepare(path.ta);
  k.prepare(path.tk);
  auto fetch = [&](int64_t at) {
    const int m = path.tokens(at);
    a.load(path.a + at * path.ta, path.ta, m, p.da);
    k.load(path.k + at * path.tk, path.tk, m, p.da);
  };
  if (path.total > 0) fetch(0);
  for (int64_t at = 0; at < path.total; at += kChunk) {
    const int64_t next = at + kChunk;
    const int m = path.tokens(at);
    __syncthreads();                                        // the chunk before has been read
    sQ.fill(a, m, p.da);
    sB.fill(k, m, p.da);
    // (c is wanted behind the next barrier but one, far enough away for its loads)
    load_c<float, FAST>(c, path.c + at * path.tc, path.tc, m, g, ccol, p.dc);
    __syncthreads();
    if (wave < 3) {                                         // a tile of A, transposed
      acc32 t = (acc32)(0.0f);
#pragma unroll
      for (int kt = 0; kt < DA / 32; ++kt) {
        bf8 x[3], y[3];
        sB.row8(16 * at_jt + lr, 32 * kt + 8 * g, x);
        sQ.row8(16 * at_it + lr, 32 * kt + 8 * g, y);
        t = mma6(x, y, t);
      }
      float v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int apart = 16 * (at_it - at_jt) + lr - 4 * g - r;
        v[r] = apart >= 0 ? t[r] * (ab * sP[apart > 0 ? apart : 0]) : 0.0f;   // a choice, not a product with 0: the term above may be a NaN
      }
      bf4 q[3];
      split(v, q);
#pragma unroll
      for (int i = 0; i < 3; ++i) *(bf4*)(sA[i] + (16 * at_it + lr) * APITCH + 8 * g + 4 * at_jt) = q[i];
    }
    acc32 o[2];
    o[0] = o[1] = (acc32)(0.0f);
#pragma unroll
    for (int kt = 0; kt < KT / 2; ++kt) {
      const float v[8] = {S[2 * kt][0], S[2 * kt][1], S[2 * kt][2], S[2 * kt][3], S[2 * kt + 1][0], S[2 * kt + 1][1], S[2 * kt + 1][2], S[2 * kt + 1][3]};
      bf8 x[3], y[3];
      sQ.row8(lr, 32 * (m0 + kt) + 8 * g, x);
      split(v, y);
      o[0] = mma6(x, y, o[0]);
      sQ.row8(16 + lr, 32 * (m0 + kt) + 8 * g, x);
      o[1] = mma6(x, y, o[1]);
    }
    // of two wavefronts on the same columns each finishes one of the tiles
    acc32 e[2 / HALVES];
    if constexpr (HALVES == 2) {
      e[0] = half ? o[1] : o[0];
      sX[wave][lane] = half ? o[0] : o[1];
    } else {
      e[0] = o[0];
      e[1] = o[1];
    }
    __syncthreads();
    if constexpr (HALVES == 2) e[0] += sX[wave ^ CT][lane];
    {
      take(c, c, m, g);
      const float v[8] = {c[0][0], c[0][1], c[0][2], c[0][3], c[1][0], c[1][1], c[1][2], c[1][3]};
      bf8 y[3];
      split(v, y);
#pragma unroll
      for (int it = 0; it < 2 / HALVES; ++it) {
        const int row = 16 * (half + it);
        bf8 x[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) x[i] = *(const bf8*)(sA[i] + (row + lr) * APITCH + 8 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r) e[it][r] *= p.scale_a * sP[row + 4 * g + r + after];
        e[it] = mma6(x, y, e[it]);
      }
    }
    if (live && m > 16 * half) put_o<float, acc32, FAST, 2 / HALVES>(e, path.o + (at + 16 * half) * path.to, path.to, m - 16 * half, g, col, p.dc);
    if (next < path.total) fetch(next);                     // (in front of A's tiles: the same time, and more registers)
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int e = m - after - (16 * jt + 4 * g + r);
        c[jt][r] *= p.scale_b * sP[e > 0 ? e : 0];
      }
    add_tokens32<DA, KT>(S, sB, c, m < kChunk ? sP[m] : next_factor(sF, debt), m0, g, lr);
  }
  // (the compiler would keep every row's offset from the loads of the first state to here, in registers the loop needs)
  int ge = g;
  asm volatile("" : "+v"(ge));
  if (!live) return;
  if (half == 0) zero_tail(p, path, g, col);
  if (p.s1 && w.segment == pl.segments - 1) {
    float* s1 = p.s1 + path.b * p.s1_b + path.h * p.s1_h + col * p.s1_c;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int d = 32 * (m0 + (kt >> 1)) + 8 * ge + 4 * (kt & 1) + r;
        if (d < p.da) s1[d * p.s1_r] = S[kt][r];
      }
  }
}

template <int DA, int WAVES, int HALVES, bool BACK, bool FAST>
__global__ __launch_bounds__(64 * WAVES, (kWaves<DA, WAVES>)) void sums_f32(Role<float> p, Plan<float> pl) {
  constexpr int KT = DA / 16 / HALVES, CT = WAVES / HALVES;
  constexpr int after = BACK ? 0 : 1;
  __shared__ __attribute__((aligned(16))) Pieces<DA> sB[2];
  __shared__ Rounded sF;                                    // e^{32 g}
  const Work w = work_of(pl, pl.slots - 1);
  if (!w.live) return;
  const Path<float, BACK> path(p, w.group, w.segment * pl.part_tokens, pl.part_tokens);
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63, g = lane >> 4, lr = lane & 15;
  const int half = HALVES == 2 ? wave / CT : 0, m0 = half * (KT / 2);
  const int col = (w.slice * CT + wave % CT) * 16 + lr;
  const int ccol = col < p.dc ? col : p.dc - 1;
  acc32 S[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt) S[kt] = (acc32)(0.0f);
  const float ld = p.log_decay[path.h];
  float wt[2][4];
  weights(wt, p.scale_b, ld, kChunk, after, g);
  if (threadIdx.x == 0) sF = rounded(power((double)ld, (int64_t)kChunk));
  float debt = 0.0f;
  Tile<float, DA, FAST, 64 * WAVES> k;
  float c[2][4], cn[2][4];
  k.prepare(path.tk);
  auto fetch = [&](int64_t at) {
    const int m = path.tokens(at);
    k.load(path.k + at * path.tk, path.tk, m, p.da);
    load_c<float, FAST>(cn, path.c + at * path.tc, path.tc, m, g, ccol, p.dc);
  };
  if (path.total > 0) fetch(0);
  int turn = 0;
  for (int64_t at = 0; at < path.total; at += kChunk, turn ^= 1) {
    const int m = path.tokens(at);
    sB[turn].fill(k, m, p.da);                              // (two buffers: one barrier a chunk)
    if (m < kChunk) weights(wt, p.scale_b, ld, m, after, g);
    take(c, cn, m, g);
#pragma unroll
    for (int jt = 0; jt < 2; ++jt)
#pragma unroll
      for (int r = 0; r < 4; ++r) c[jt][r] *= wt[jt][r];
    __syncthreads();
    if (at + kChunk < path.total) fetch(at + kChunk);
    add_tokens32<DA, KT>(S, sB[turn], c, m < kChunk ? power(ld, (int64_t)m) : next_factor(sF, debt), m0, g, lr);
  }
  if (col >= p.dc) return;
  float* s1 = pl.states + ((int64_t)w.group * pl.slots + w.segment + 1) * p.da * p.dc + col;
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int d = 32 * (m0 + (kt >> 1)) + 8 * g + 4 * (kt & 1) + r;
      if (d < p.da) s1[(int64_t)d * p.dc] = S[kt][r];
    }
}

// Tokens in front of a slot, of a sequence of n.
template <typename T> __device__ __forceinline__ int64_t tokens_before(const Plan<T>& pl, int64_t n, int slot) {
  const int64_t t = slot * pl.part_tokens;
  return t < n ? t : n;
}

// From slot to slot: whole parts, then what is left of the sequence, then nothing.
template <typename T> struct Decays {
  int64_t n, part;
  T whole, rest;
  Rounded split;
  float debt;
  __device__ __forceinline__ Decays(const Plan<T>& pl, T ld, int64_t n_) : n(n_), part(pl.part_tokens), debt(0.0f) {
    const double e = power((double)ld, part);
    whole = (T)e;
    split = rounded(e);
    rest = power(ld, n % part);
  }
  __device__ __forceinline__ T into(int slot) {
    const int64_t before = (int64_t)(slot - 1) * part;
    if (before + part <= n) {
      if constexpr (sizeof(T) == 4) return next_factor(split, debt);
      else return whole;
    }
    return before < n ? rest : (T)1;
  }
};

// From the parts' shares to the states in front of the segments (the slots at multiples of `parts`): a lane takes V neighbouring
// elements of a head's state, BATCH slots on their way at a time (no load may pass the stores of the batch before).
template <typename T, int V, int BATCH>
__device__ __forceinline__ void carry(T* at, int64_t per, int& k, T (&s)[V], Decays<T>& decays, const Plan<T>& pl) {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  vec_t v[BATCH];
#pragma unroll
  for (int u = 0; u < BATCH; ++u) v[u] = *(const vec_t*)(at + (int64_t)(k + u < pl.slots ? k + u : pl.slots - 1) * per);
#pragma unroll
  for (int u = 0; u < BATCH; ++u) {
    if (k + u >= pl.slots) break;
    const T f = decays.into(k + u);
    vec_t to;
#pragma unroll
    for (int e = 0; e < V; ++e) to[e] = s[e] = s[e] * f + v[u][e];
    if ((k + u) % pl.parts == 0) *(vec_t*)(at + (int64_t)(k + u) * per) = to;
  }
  k += BATCH;
}

template <typename T, int V>
__global__ __launch_bounds__(256) void segment_states(Role<T> p, Plan<T> pl) {
  const int per = p.da * p.dc;
  const int blocks = (per + 256 * V - 1) / (256 * V);
  const int group = (int)(blockIdx.x / (unsigned)blocks);
  const int i = ((int)(blockIdx.x - (unsigned)group * (unsigned)blocks) * 256 + (int)threadIdx.x) * V;
  if (i >= per) return;
  const int64_t b = group / (int)p.heads;
  const int h = (int)(group - b * p.heads);
  const int64_t n = length_of(p, b);
  const T ld = p.log_decay[h];
  const int r = i / p.dc, c = i - r * p.dc;
  T* at = pl.states + (int64_t)group * pl.slots * per + i;
  T s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s[e] = p.s0 ? p.s0[b * p.s0_b + h * p.s0_h + r * p.s0_r + (c + e) * p.s0_c] : (T)0;
    at[e] = s[e];
  }
  Decays<T> decays(pl, ld, n);
  int k = 1;
  while (k < pl.slots) carry<T, V, 8>(at, per, k, s, decays, pl);
}

// The same for few states, where the length of the chain counts: a lane takes one element, and the four wavefronts of a
// workgroup a quarter of up to 4 MOST slots each. They add up theirs, exchange the sums and add what lies in front.
template <typename T, int MOST>
__device__ __forceinline__ void carry_quarters(T* at, int64_t per, int from, int count, T& s, T ld, int64_t n, const Plan<T>& pl, bool live, T (&sums)[4][64]) {
  const int wave = (int)threadIdx.x >> 6, lane = (int)threadIdx.x & 63;
  const int each = (count + 3) / 4;
  auto first = [&](int w) { const int k = w * each; return from + (k < count ? k : count); };
  auto decay = [&](int lo, int hi) { return power(ld, tokens_before(pl, n, hi) - tokens_before(pl, n, lo)); };   // from slot to slot
  const int lo = first(wave), hi = first(wave + 1);
  T v[MOST], t = (T)0;
#pragma unroll
  for (int u = 0; u < MOST; ++u) v[u] = at[(int64_t)(lo + u < pl.slots ? lo + u : pl.slots - 1) * per];
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    if (lo + u >= hi) break;
    v[u] = t = t * decay(lo + u - 1, lo + u) + v[u];
  }
  __syncthreads();
  sums[wave][lane] = t;
  __syncthreads();
  T in = s;                                                 // the state in front of this quarter
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w == wave) in = s;
    if (first(w) < first(w + 1)) s = s * decay(first(w) - 1, first(w + 1) - 1) + sums[w][lane];
  }
#pragma unroll
  for (int u = 0; u < MOST; ++u) {
    if (lo + u >= hi) break;
    if ((lo + u) % pl.parts == 0 && live) at[(int64_t)(lo + u) * per] = v[u] + in * decay(lo - 1, lo + u);
  }
}

template <typename T>
__global__ __launch_bounds__(256) void segment_states_few(Role<T> p, Plan<T> pl) {
  __shared__ T sums[4][64];
  const int per = p.da * p.dc;
  const int blocks = (per + 63) / 64;
  const int group = (int)(blockIdx.x / (unsigned)blocks);
  int i = (int)(blockIdx.x - (unsigned)group * (unsigned)blocks) * 64 + ((int)threadIdx.x & 63);
  const bool live = i < per;
  if (!live) i = 0;
  const int64_t b = group / (int)p.heads;
  const int h = (int)(group - b * p.heads);
  const int64_t n = length_of(p, b);
  const T ld = p.log_decay[h];
  const int r = i / p.dc, c = i - r * p.dc;
  T* at = pl.states + (int64_t)group * pl.slots * per + i;
  T s = p.s0 ? p.s0[b * p.s0_b + h * p.s0_h + r * p.s0_r + c * p.s0_c] : (T)0;
  if (live && threadIdx.x < 64) at[0] = s;
  for (int k = 1; k < pl.slots; k += 128) {
    const int count = pl.slots - k < 128 ? pl.slots - k : 128;
    if (count <= 16) carry_quarters<T, 4>(at, per, k, count, s, ld, n, pl, live, sums);
    else carry_quarters<T, 32>(at, per, k, count, s, ld, n, pl, live, sums);
  }
}

static int workgroups_per_cu(const void* kernel, int threads) {
  int n = 0;
  if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, threads, 0) != hipSuccess || n < 1) { (void)hipGetLastError(); n = 1; }
  return n;
}

template <typename T> using Kernel = void (*)(Role<T>, Plan<T>);

// The states in front of the segments of one walk. The two backward roles of a backward pass walk the same keys and values
// with their parts exchanged, so the second reads the first's states transposed.
template <typename T> struct Segments {
  Plan<T> plan = {};
  Scratch states;
  bool made = false;
};

// A wavefront takes 16 columns.
template <typename T, Kernel<T> CHUNKS, Kernel<T> SUMS>
static int run_chunks(const Role<T>& p, Segments<T>& seg, int waves, int cols) {
  const dim3 block((unsigned)(64 * waves));
  Plan<T>& pl = seg.plan;
  pl.slices = (p.dc + cols - 1) / cols;
  if (seg.made) {
    pl.st_r = 1; pl.st_c = p.da;
  } else {
    pl.groups = (int)(p.batch * p.heads);
    pl.st_r = p.dc; pl.st_c = 1;
    const int64_t wgs = (int64_t)pl.groups * pl.slices;
    const int64_t n_chunks = (p.tokens + kChunk - 1) / kChunk;
    // As many segments as the device has room for workgroups, up to two of eight wavefronts or three of four on a CU (more
    // win nothing: 32 x 1024 tokens, 16 heads of 64 x 64 in one segment, two workgroups a CU, take 124 us, in two segments
    // 173); a segment has two chunks at least.
    static const int room = workgroups_per_cu((const void*)CHUNKS, 64 * waves), sums_room = workgroups_per_cu((const void*)SUMS, 64 * waves);
    const int a_cu = waves == 8 ? 2 : 3;
    int64_t segments = (int64_t)(room < a_cu ? room : a_cu) * num_cus() / wgs;
    if (segments > n_chunks / 2) segments = n_chunks / 2;
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
    if (pl.segments > 1) {
      AM_TRY(seg.states.take((size_t)pl.groups * pl.slots * p.da * p.dc * sizeof(T)));
      pl.states = (T*)seg.states.p;
      const int64_t ids = ((int64_t)pl.groups * (pl.slots - 1) + 7) / 8 * 8 * pl.slices;
      hipLaunchKernelGGL(SUMS, dim3((unsigned)ids), block, 0, stream(), p, pl);
      AM_TRY(check_launch("decay attention: sums"));
      // Vectors of 16 bytes and one walk over the slots where that still makes a wavefront a CU: 64 states of 128 x 128 and 8
      // slots, 62 MB, 21.5 us in single elements, 11.9 in vectors; in quarters the whole call takes 225 us in place of 216. Below,
      // quarters: 8 states of 64 x 64 and 86 slots, the whole call 67 us in one walk, 62 in quarters.
      constexpr int V = 16 / (int)sizeof(T);
      const int per = p.da * p.dc;
      if ((int64_t)pl.groups * per / V < (int64_t)64 * num_cus())
        hipLaunchKernelGGL((segment_states_few<T>), dim3((unsigned)(pl.groups * ((per + 63) / 64))), dim3(256), 0, stream(), p, pl);
      else if (p.dc % V == 0)
        hipLaunchKernelGGL((segment_states<T, V>), dim3((unsigned)(pl.groups * ((per + 256 * V - 1) / (256 * V)))), dim3(256), 0, stream(), p, pl);
      else
        hipLaunchKernelGGL((segment_states<T, 1>), dim3((unsigned)(pl.groups * ((per + 255) / 256))), dim3(256), 0, stream(), p, pl);
      AM_TRY(check_launch("decay attention: states"));
    }
    seg.made = true;
  }
  const int64_t ids = ((int64_t)pl.groups * pl.segments + 7) / 8 * 8 * pl.slices;
  hipLaunchKernelGGL(CHUNKS, dim3((unsigned)ids), block, 0, stream(), p, pl);
  return check_launch("decay attention: chunks");
}

template <int DA, bool BACK, bool FAST> static int run_sized(const Role<double>& p, Segments<double>& seg) {
  return run_chunks<double, chunks_f64<DA, BACK, FAST>, sums_f64<DA, BACK, FAST>>(p, seg, kWaves64, kCols64);
}
// Eight wavefronts where there are more than 64 columns (a and b are then split and staged once for all), unless the workgroups
// of 128 columns leave CUs without work however short their segments.
template <int DA, bool BACK, bool FAST> static int run_sized(const Role<float>& p, Segments<float>& seg) {
  const int64_t pairs = (p.tokens + 2 * kChunk - 1) / (2 * kChunk);
  const bool wide = p.dc > 64 && p.batch * p.heads * ((p.dc + 127) / 128) * (pairs > 1 ? pairs : 1) >= num_cus();
  if (wide) return run_chunks<float, chunks_f32<DA, 8, 1, BACK, FAST>, sums_f32<DA, 8, 1, BACK, FAST>>(p, seg, 8, 128);
  // 64 columns: from 128 rows on the rows are halved, and twice as many wavefronts share a workgroup's LDS. 8 x 1024 tokens, 8 heads
  // of 192 x 64: 82 -> 67 us, of 128 x 64: 52 either way, 8 x 64 tokens, 16 heads of 128 x 128: 15 -> 13; with 64 rows 32 x 1024
  // tokens, 16 heads of 64 x 64 lose: 126 -> 137.
  if constexpr (DA % 64 == 0 && DA >= 128) return run_chunks<float, chunks_f32<DA, 8, 2, BACK, FAST>, sums_f32<DA, 8, 2, BACK, FAST>>(p, seg, 8, 64);
  else return run_chunks<float, chunks_f32<DA, 4, 1, BACK, FAST>, sums_f32<DA, 4, 1, BACK, FAST>>(p, seg, 4, 64);
}

template <bool BACK, bool FAST, typename T> static int run_fast(const Role<T>& p, Segments<T>& seg) {
  if (p.da <= 32) return run_sized<32, BACK, FAST>(p, seg);
  if (p.da <= 64) return run_sized<64, BACK, FAST>(p, seg);
  if (p.da <= 96) return run_sized<96, BACK, FAST>(p, seg);
  if (p.da <= 128) return run_sized<128, BACK, FAST>(p, seg);
  if (p.da <= 192) return run_sized<192, BACK, FAST>(p, seg);
  return run_sized<256, BACK, FAST>(p, seg);
}

template <typename T, bool BACK>
static int run_role(const Role<T>& p, Segments<T>& seg) {
  // FAST: rows of whole vectors, and 32 tokens of every operand within 2^31 bytes
  const int64_t most = ((int64_t)1 << 31) / (kChunk * (int64_t)sizeof(T)) - kMostDim;
  auto near = [&](int64_t t) { return t < most && -t < most; };
  const bool fast = p.da % (16 / (int)sizeof(T)) == 0 && near(p.a.t) && near(p.b.t) && near(p.c.t) && near(p.o_t);
  return fast ? run_fast<BACK, true>(p, seg) : run_fast<BACK, false>(p, seg);
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

// NT: the states go past the caches both ways, where they are larger than those keep (192 sequences, 16 heads of 128 x 128:
// 83.8 -> 77.2 us, 4.8 -> 5.2 TB/s; with the loads alone 82.6). Single elements (rows that are no whole vectors) go through them at
// any size: past them is not measured; heads of 126 x 126 take 84.9 us, 4.6 TB/s, of 127 x 127 in float64 5.1 TB/s.
template <typename T, int V, bool NT>
__global__ __launch_bounds__(256) void step(StepArgs<T> p, int lanes, int tiles) {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  __shared__ T fold[256 * V];
  const int64_t head = blockIdx.x / tiles;
  const int tile = (int)(blockIdx.x - head * tiles);
  const int64_t b = head / p.heads;
  const int h = (int)(head - b * p.heads);
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
      vec_t* at = (vec_t*)(s + (int64_t)r * p.dv);
      vec_t w;
      if constexpr (NT) w = __builtin_nontemporal_load(at);
      else w = *at;
      w = w * lam + v * k[r];
      acc += w * q[r];
      if constexpr (NT) __builtin_nontemporal_store(w, at);
      else *at = w;
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
template <typename T> static bool broadcast_result(const Result<T>& r, int64_t batch, int64_t tokens, int64_t heads, int64_t width) {
  return tokens > 0 && ((batch > 1 && r.b == 0) || (tokens > 1 && r.t < width && -r.t < width) || (heads > 1 && r.h == 0));
}
// Any token stride will do for a single token, but the chunks write whole tiles of rows and leave it to the buffer's end to drop
// those behind the last token: a row's width at least has to lie between them.
template <typename T> static void one_token(Result<T>& r, int64_t tokens, int64_t width) {
  if (tokens == 1) r.t = width;
}

template <typename T>
static int forward(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale,
                   const T* log_decay, const int64_t* lengths, Strided<T> q, Strided<T> k, Strided<T> v, const T* s0, int64_t s0_b,
                   int64_t s0_h, Result<T> out, T* s1, int64_t s1_b, int64_t s1_h) {
  AM_TRY(check_sizes(fn, batch, tokens, heads, kv_heads, dk, dv));
  if (batch == 0 || heads == 0) return AM_OK;
  if (!log_decay || (tokens && (!q.p || !k.p || !v.p || !out.p))) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if (broadcast_result(out, batch, tokens, heads, dv) || (s1 && ((batch > 1 && s1_b == 0) || (heads > 1 && s1_h == 0))))
    return fail(AM_E_SHAPE, "%s: a result is a broadcast view, or its tokens overlap", fn);
  one_token(out, tokens, dv);
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
  Segments<T> seg;
  return run_role<T, false>(p, seg);
}

// out[b, t, head, :] = the sum of the `group` heads' shares that follow each other, in the heads' order
template <typename T, int V>
__global__ __launch_bounds__(256) void fold(const T* shares, Result<T> out, int64_t first, int64_t rows, int tokens, int kv_heads, int group, int d) {
  typedef T vec_t __attribute__((ext_vector_type(V)));
  const int per = d / V;
  const int64_t i = (first + blockIdx.x) * 256 + threadIdx.x;
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
  if (tokens >= ((int64_t)1 << 31)) return fail(AM_E_SHAPE, "decay attention: too many tokens for shared heads");
  constexpr int64_t kLaunch = (int64_t)1 << 16;             // workgroups: a launch has less than 2^32 threads
  for (int64_t first = 0; first < wgs; first += kLaunch) {
    const dim3 grid((unsigned)(wgs - first < kLaunch ? wgs - first : kLaunch)), block(256);
    if (vec) hipLaunchKernelGGL((fold<T, W>), grid, block, 0, stream(), shares, out, first, rows, (int)tokens, (int)kv_heads, group, d);
    else hipLaunchKernelGGL((fold<T, 1>), grid, block, 0, stream(), shares, out, first, rows, (int)tokens, (int)kv_heads, group, d);
    AM_TRY(check_launch("fold"));
  }
  return AM_OK;
}

template <typename T>
static int backward(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv, T scale,
                    const T* log_decay, const int64_t* lengths, Strided<T> go, Strided<T> q, Strided<T> k, Strided<T> v, const T* s0,
                    int64_t s0_b, int64_t s0_h, const T* gs, int64_t gs_b, int64_t gs_h, Result<T> dq, Result<T> dkey, Result<T> dval,
                    T* gs0, int64_t gs0_b, int64_t gs0_h) {
  AM_TRY(check_sizes(fn, batch, tokens, heads, kv_heads, dk, dv));
  if (batch == 0 || heads == 0) return AM_OK;
  if (!log_decay || (tokens && (!go.p || !q.p || !k.p || !v.p || !dq.p || !dkey.p || !dval.p))) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if (broadcast_result(dq, batch, tokens, heads, dk) || broadcast_result(dkey, batch, tokens, kv_heads, dk) ||
      broadcast_result(dval, batch, tokens, kv_heads, dv) ||
      (gs0 && ((batch > 1 && gs0_b == 0) || (heads > 1 && gs0_h == 0))))
    return fail(AM_E_SHAPE, "%s: a result is a broadcast view, or its tokens overlap", fn);
  one_token(dq, tokens, dk);
  one_token(dkey, tokens, dk);
  one_token(dval, tokens, dv);
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
  {
    Segments<T> seg;
    AM_TRY((run_role<T, false>(p, seg)));
  }
  // dk and dv: backwards. Where heads share a key / value head each writes its own share, and `fold_heads` adds them up.
  // dk first: dv's walk writes the first state's gradient, which may lie over the last state's.
  p.scale_a = (T)1; p.scale_b = scale;
  p.s0 = gs; p.s0_b = gs_b; p.s0_h = gs_h;
  Segments<T> seg;
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
  AM_TRY((run_role<T, true>(p, seg)));
  if (group > 1) AM_TRY(fold_heads((const T*)shares.p, dkey, batch, tokens, kv_heads, group, (int)dk));
  p.a = K; p.b = Q; p.c = G;
  into(dval, dv);
  p.s0_r = dv; p.s0_c = 1;
  p.s1 = gs0; p.s1_b = gs0_b; p.s1_h = gs0_h; p.s1_r = dv; p.s1_c = 1;
  p.da = (int)dk; p.dc = (int)dv;
  AM_TRY((run_role<T, true>(p, seg)));
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
  const bool nt = (double)batch * heads * dk * dv * sizeof(T) > nt_threshold_bytes();
  if (vec && nt) hipLaunchKernelGGL((step<T, W, true>), dim3((unsigned)wgs), dim3(256), 0, stream(), p, lanes, tiles);
  else if (vec) hipLaunchKernelGGL((step<T, W, false>), dim3((unsigned)wgs), dim3(256), 0, stream(), p, lanes, tiles);
  else hipLaunchKernelGGL((step<T, 1, false>), dim3((unsigned)wgs), dim3(256), 0, stream(), p, lanes, tiles);
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
