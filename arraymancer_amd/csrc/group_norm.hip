// Group normalisation with an activation over channels-last tensors: am_hip_group_norm_*, am_hip_group_norm_backward_*.
//
// x [batch, spatial, channels]; the channels form `groups` groups of `per`, and each (sample, group) is normalised over its
// spatial * per elements:
//     xhat = (x - mean) * rstd      z = xhat * weight[c] + bias[c]      y = act(z)
// Backwards, with dz = dy * act'(z) and averages over the same elements,
//     dx = rstd * (weight dz - avg(weight dz) - xhat * avg(weight dz xhat))
//     dweight[c] = sum dz xhat      dbias[c] = sum dz                       (over batch and spatial)
//
// Three ways through it:
//  - `team_*`: the elements of a group fit the registers of a team of lanes (8 .. 64, or a workgroup of 256). One launch,
//    x is read once, mean and squared deviations are two folds over registers. A team keeps its group and walks over samples,
//    with the group's parameters in registers; backwards it also adds up its lanes' shares of dweight and dbias on the way.
//  - `image_*`: many rows, whose group fits the registers of a workgroup of up to 1024 lanes, in runs of memory that are not too short. As the teams do it: one launch, every tensor moves once (backwards the activation is computed once too).
//  - slabs, for the rest: a workgroup takes a slab of rows of one sample and reads them whole, channels next to each other, whatever the
//    group's width; a lane owns V channels and keeps two sums for each. The slabs' sums per channel go to scratch memory
//    and a small kernel folds them in a fixed order, per group (mean, rstd, or the two averages of the backward pass) and,
//    backwards, per channel; then a second pass over the slabs writes the result. The forward pass keeps means and squared
//    deviations from them, in double, never sums of squares about a fixed point: nothing cancels where the mean is large
//    against the deviation, or where single elements (an image's empty border) lie far from the rest.
#include "common.h"
#include "fastdiv.h"
#include "scratch.h"

namespace am {
namespace gnorm {

template <typename T> struct Args {
  const T* x; int64_t x_n, x_s;
  const T* dy; int64_t dy_n, dy_s;
  const T* weight; const T* bias;
  T* y; int64_t y_n, y_s;            // forward: the result; backward: dx
  T* mean; T* rstd;                  // [batch, groups]
  T* dweight; T* dbias;
  double* part;                      // slabs: [n][slab][channel][2]: forward mean and squared deviations, backward sums of dz xhat and dz
  double* chan;                      // slabs, backward: [n][channel][2], null when no parameter's gradient is wanted
  T* share;                          // teams, backward: [slot][group][row][channel of the group][2] (workgroups: rows summed), null likewise
  T* coef;                           // backward: [n][group][2], the two averages
  T eps;
  int64_t batch, spatial;
  int channels, groups, per;
  int64_t n0, nc;                    // samples of this launch: n0 .. n0 + nc
  int slabs; int64_t rows_per_slab;
  int folds;                         // slabs, backward: the first so many workgroups of the second pass fold the parameters' gradients
  int tiles, lanes, rows_at_once;    // channel tiles; lanes per row of a tile; rows a workgroup reads at once
  FastDiv per_div, tiles_div, slabs_div, groups_div, units_div;
};

__device__ __forceinline__ float dev_rsqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double dev_rsqrt(double v) { return 1.0 / sqrt(v); }

// 1 / (1 + e^-z). In float from the hardware's exp2 and reciprocal, one step each: -z log2(e) is split into the product
// and what its rounding lost, so that the error does not grow with z (4 steps in all). The backward pass over a large image
// spends most of its instructions here; expf and a division take three times as many. Where exp2 leaves the range there is
// nothing to correct (and an infinite z has no rounding to take a difference of).
__device__ __forceinline__ float sigmoid(float z) {
  const float hi = z * -1.44269504f;
  const float lo = fmaf(z, -1.44269504f, -hi) + z * -1.92596299e-8f;
  const float corr = fabsf(hi) < 127.0f ? 1.0f + lo * 0.693147181f : 1.0f;
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(hi) * corr);
}
__device__ __forceinline__ double sigmoid(double z) { return 1.0 / (1.0 + exp(-z)); }

template <typename T, int ACT> __device__ __forceinline__ T activate(T z) {
  if constexpr (ACT == AM_ACT_RELU) return ((T)0 >= z) ? (T)0 : z;
  else if constexpr (ACT == AM_ACT_SILU) return z * sigmoid(z);
  else return z;
}
// dy * act'(z)
template <typename T, int ACT> __device__ __forceinline__ T through(T dy, T z) {
  if constexpr (ACT == AM_ACT_RELU) return ((T)0 >= z) ? (T)0 : dy;
  else if constexpr (ACT == AM_ACT_SILU) {
    const T s = sigmoid(z);
    return dy * (s * ((T)1 + z * ((T)1 - s)));
  } else return dy;
}

// NT: past the caches, for the last reading of a tensor larger than they keep.
template <bool NT, typename V> __device__ __forceinline__ V fetch(const V* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

template <typename T, int V> struct Vec { typedef T type __attribute__((ext_vector_type(V))); };

// Sum over the lanes of a team: butterflies within a wavefront, then (WIDE: the team is the workgroup of four) through LDS.
template <typename T, bool WIDE> __device__ __forceinline__ T team_sum(T v, int lanes, T* lds) {
  for (int d = (WIDE ? 64 : lanes) >> 1; d >= 1; d >>= 1) v += __shfl_xor(v, d, 64);
  if constexpr (WIDE) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (lds[0] + lds[1]) + (lds[2] + lds[3]);
  }
  return v;
}

constexpr int kUnits = 8;   // units (vectors) a lane of a team holds at most

// A team's place: its group, the first sample it takes, and its lanes' units (q = lane + k * lanes): row q / units-per-row of
// the sample, channels V * (q % units-per-row) ... of the group. Units behind the last repeat it, so that every load is
// unconditional; they count for nothing and are not written.
template <typename T, int V, int U, bool WIDE> struct Team {
  int j0, step, g;
  int64_t slot;
  bool there, live[U];
  uint32_t row[U], col[U];
  __device__ __forceinline__ Team(const Args<T>& p, int lanes, int units, int64_t slots) {
    const int teams = WIDE ? 1 : 256 / lanes;
    const int64_t team = (int64_t)blockIdx.x * teams + (WIDE ? 0 : (int)threadIdx.x / lanes);
    j0 = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (lanes - 1);
    step = WIDE ? 256 : lanes;
    slot = team / p.groups;
    g = (int)(team - slot * p.groups);
    there = slot < slots;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      int q = j0 + k * step;
      live[k] = q < units;
      q = live[k] ? q : units - 1;
      row[k] = p.units_div.divmod((uint32_t)q, col[k]);
      col[k] *= V;
    }
  }
};

template <typename T, int V, int U, bool WIDE, int ACT, bool NT>
__global__ __launch_bounds__(256) void team_forward(Args<T> p, int lanes, int units, int64_t slots) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ T lds[4];
  const Team<T, V, U, WIDE> t(p, lanes, units, slots);
  if (!t.there) return;       // whole teams leave together, and teams never straddle a wavefront
  const int c0 = t.g * p.per;
  vec_t w[U], b[U];
#pragma unroll
  for (int k = 0; k < U; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[k][e] = p.weight ? p.weight[c0 + t.col[k] + e] : (T)1;
      b[k][e] = p.bias ? p.bias[c0 + t.col[k] + e] : (T)0;
    }
  const T count = (T)((T)p.spatial * (T)p.per);
  for (int64_t n = t.slot; n < p.batch; n += slots) {
    const T* x = p.x + n * p.x_n + c0;
    vec_t v[U];
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = fetch<NT>((const vec_t*)(x + t.row[k] * p.x_s + t.col[k]));
    T sum = (T)0;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) sum += t.live[k] ? v[k][e] : (T)0;
    const T mean = team_sum<T, WIDE>(sum, lanes, lds) / count;
    T sq = (T)0;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[k][e] -= mean;
        sq += t.live[k] ? v[k][e] * v[k][e] : (T)0;
      }
    const T rstd = dev_rsqrt(team_sum<T, WIDE>(sq, lanes, lds) / count + p.eps);
    if (t.j0 == 0 && p.mean) { p.mean[n * p.groups + t.g] = mean; p.rstd[n * p.groups + t.g] = rstd; }
    T* y = p.y + n * p.y_n + c0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      vec_t out;
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = activate<T, ACT>(v[k][e] * rstd * w[k][e] + b[k][e]);
      if (t.live[k]) *(vec_t*)(y + t.row[k] * p.y_s + t.col[k]) = out;
    }
  }
}

template <typename T, int V, int U, bool WIDE, int ACT, bool NT>
__global__ __launch_bounds__(256) void team_backward(Args<T> p, int lanes, int units, int64_t slots) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ T lds[4];
  const Team<T, V, U, WIDE> t(p, lanes, units, slots);
  if (!t.there) return;
  const int c0 = t.g * p.per;
  vec_t w[U], b[U], dw[U], db[U];
#pragma unroll
  for (int k = 0; k < U; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[k][e] = p.weight ? p.weight[c0 + t.col[k] + e] : (T)1;
      b[k][e] = p.bias ? p.bias[c0 + t.col[k] + e] : (T)0;
      dw[k][e] = db[k][e] = (T)0;
    }
  const T count = (T)((T)p.spatial * (T)p.per);
  for (int64_t n = t.slot; n < p.batch; n += slots) {
    const T* x = p.x + n * p.x_n + c0;
    const T* dy = p.dy + n * p.dy_n + c0;
    const T mean = p.mean[n * p.groups + t.g], rstd = p.rstd[n * p.groups + t.g];
    vec_t h[U], d[U];     // xhat and weight * dz
#pragma unroll
    for (int k = 0; k < U; ++k) {
      h[k] = fetch<NT>((const vec_t*)(x + t.row[k] * p.x_s + t.col[k]));
      d[k] = fetch<NT>((const vec_t*)(dy + t.row[k] * p.dy_s + t.col[k]));
    }
    T s1 = (T)0, s2 = (T)0;
#pragma unroll
    for (int k = 0; k < U; ++k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        h[k][e] = (h[k][e] - mean) * rstd;
        const T dz = through<T, ACT>(d[k][e], h[k][e] * w[k][e] + b[k][e]);
        dw[k][e] += dz * h[k][e];
        db[k][e] += dz;
        d[k][e] = dz * w[k][e];
        s1 += t.live[k] ? d[k][e] : (T)0;
        s2 += t.live[k] ? d[k][e] * h[k][e] : (T)0;
      }
    s1 = team_sum<T, WIDE>(s1, lanes, lds) / count;
    s2 = team_sum<T, WIDE>(s2, lanes, lds) / count;
    T* dx = p.y + n * p.y_n + c0;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      vec_t out;
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = rstd * (d[k][e] - s1 - h[k][e] * s2);
      if (t.live[k]) *(vec_t*)(dx + t.row[k] * p.y_s + t.col[k]) = out;
    }
  }
  if (!p.share) return;
  if constexpr (WIDE) {
    // a workgroup adds up the rows of its group first, a lane staying with one channel
    __shared__ T rows[256 * U * V];
    __shared__ T part[256];
    const int wide = p.per < 256 ? p.per : 256, over = 256 / wide, k0 = (int)threadIdx.x / wide, cl = (int)threadIdx.x - k0 * wide;
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (t.live[k])
#pragma unroll
          for (int e = 0; e < V; ++e) rows[(t.j0 + k * 256) * V + e] = which ? db[k][e] : dw[k][e];
      __syncthreads();
      for (int b0 = 0; b0 < p.per; b0 += wide) {
        const int c = b0 + cl;
        const bool mine = k0 < over && c < p.per;
        T sum = (T)0;
        if (mine)
          for (int r = k0; r < (int)p.spatial; r += over) sum += rows[r * p.per + c];
        __syncthreads();
        part[threadIdx.x] = sum;
        __syncthreads();
        if (mine && k0 == 0) {
          for (int r = 1; r < over; ++r) sum += part[threadIdx.x + r * wide];
          p.share[((t.slot * p.groups + t.g) * p.per + c) * 2 + which] = sum;
        }
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      if (!t.live[k]) continue;
      T* at = p.share + (((t.slot * p.groups + t.g) * p.spatial + t.row[k]) * p.per + t.col[k]) * 2;
#pragma unroll
      for (int e = 0; e < V; ++e) { at[2 * e] = dw[k][e]; at[2 * e + 1] = db[k][e]; }
    }
  }
}

// ---- groups of an image in the registers of a workgroup ----
// Bound by memory, and by the reductions between reading and writing that nothing overlaps: a CU has registers for one
// workgroup of 1024 lanes (128 registers each; forwards fewer), for two of 512, four of 256. [128, 24, 24, 512] in 16 groups: 302 MB
// forwards in 63 us, 453 MB backwards in 101 with 512 lanes, in 139 with 1024.
constexpr int kImage = 1024;                   // lanes at most
template <typename T> constexpr int kImageHeld = 192 / (int)sizeof(T);   // elements of a tensor that a lane holds at most

// A sample's rows, channels of one group, as a buffer: the hardware adds a lane's 32-bit offset, and what lies behind the last
// row reads as 0 and is not written.
template <typename T> __device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const T* p, int64_t spatial, int64_t step, int per) {
  return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, (int)(((spatial - 1) * step + per) * (int64_t)sizeof(T)), 0x00020000);
}
template <typename V> __device__ __forceinline__ V get(__amdgpu_buffer_rsrc_t r, uint32_t off) {
  if constexpr (sizeof(V) == 4) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0));
  else if constexpr (sizeof(V) == 8) return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
  else return __builtin_bit_cast(V, __builtin_amdgcn_raw_buffer_load_b128(r, (int)off, 0, 0));
}
template <typename V> __device__ __forceinline__ void put(__amdgpu_buffer_rsrc_t r, uint32_t off, V v) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  typedef unsigned u4 __attribute__((ext_vector_type(4)));
  if constexpr (sizeof(V) == 4) __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, v), r, (int)off, 0, 0);
  else if constexpr (sizeof(V) == 8) __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, v), r, (int)off, 0, 0);
  else __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, v), r, (int)off, 0, 0);
}

// The sums of two values over the workgroup, the same in every lane.
template <typename T, int WAVES> __device__ __forceinline__ void image_sums(T& a, T& b, T (&lds)[2][WAVES]) {
  for (int d = 32; d >= 1; d >>= 1) { a += __shfl_xor(a, d, 64); b += __shfl_xor(b, d, 64); }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) { lds[0][threadIdx.x >> 6] = a; lds[1][threadIdx.x >> 6] = b; }
  __syncthreads();
  T s[2][4] = {};
#pragma unroll
  for (int i = 0; i < WAVES; ++i) { s[0][i & 3] += lds[0][i]; s[1][i & 3] += lds[1][i]; }
  a = (s[0][0] + s[0][1]) + (s[0][2] + s[0][3]);
  b = (s[1][0] + s[1][1]) + (s[1][2] + s[1][3]);
}

// A workgroup's place: workgroups that run together on a die take neighbouring groups, which share cache lines. A lane stays
// with V channels (c) and takes rows row, row + rows_at_once, ...
template <typename T, int V> struct Image {
  int64_t n;
  int g, row;
  uint32_t c;
  bool there, live;
  __device__ __forceinline__ Image(const Args<T>& p) {
    const uint32_t all = (uint32_t)(p.batch * p.groups), each = (all + 7) / 8;
    const uint32_t item = (blockIdx.x & 7) * each + (blockIdx.x >> 3);
    there = (blockIdx.x >> 3) < each && item < all;
    uint32_t gi;
    n = p.groups_div.divmod(item, gi);
    g = (int)gi;
    row = (int)p.units_div.divmod(threadIdx.x, c);
    c *= V;
    live = row < p.rows_at_once;
  }
  // a lane without rows reads and writes behind the last one
  __device__ __forceinline__ uint32_t first(int64_t step) const { return live ? (uint32_t)((row * step + c) * (int64_t)sizeof(T)) : 0x7fffffffu & ~15u; }
};

template <typename T, int LANES, int V, int U, int ACT>
__global__ __launch_bounds__(LANES, 4) void image_forward(Args<T> p) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ T lds[2][LANES / 64];
  const Image<T, V> t(p);
  if (!t.there) return;
  const int c0 = t.g * p.per, spatial = (int)p.spatial;
  vec_t v[U];
  {
    const __amdgpu_buffer_rsrc_t x = rows_of(p.x + t.n * p.x_n + c0, p.spatial, p.x_s, p.per);
    const uint32_t first = t.first(p.x_s), step = (uint32_t)(p.rows_at_once * p.x_s * (int64_t)sizeof(T));
#pragma unroll
    for (int k = 0; k < U; ++k) v[k] = get<vec_t>(x, first + (uint32_t)k * step);
  }
  T w[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    w[e] = p.weight ? p.weight[c0 + t.c + e] : (T)1;
    b[e] = p.bias ? p.bias[c0 + t.c + e] : (T)0;
  }
  const T count = (T)((T)p.spatial * (T)p.per);
  T part[4] = {}, none = (T)0;                 // four short sums in a lane
#pragma unroll
  for (int k = 0; k < U; ++k)
#pragma unroll
    for (int e = 0; e < V; ++e) part[(k * V + e) & 3] += v[k][e];
  T sum = (part[0] + part[1]) + (part[2] + part[3]);
  image_sums(sum, none, lds);
  const T mean = sum / count;
#pragma unroll
  for (int i = 0; i < 4; ++i) part[i] = (T)0;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool is = t.live && t.row + k * p.rows_at_once < spatial;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[k][e] -= mean;
      part[(k * V + e) & 3] += is ? v[k][e] * v[k][e] : (T)0;
    }
  }
  T sq = (part[0] + part[1]) + (part[2] + part[3]);
  image_sums(sq, none, lds);
  const T rstd = dev_rsqrt(sq / count + p.eps);
  if (threadIdx.x == 0 && p.mean) { p.mean[t.n * p.groups + t.g] = mean; p.rstd[t.n * p.groups + t.g] = rstd; }
  const __amdgpu_buffer_rsrc_t y = rows_of(p.y + t.n * p.y_n + c0, p.spatial, p.y_s, p.per);
  const uint32_t first = t.first(p.y_s), step = (uint32_t)(p.rows_at_once * p.y_s * (int64_t)sizeof(T));
#pragma unroll
  for (int k = 0; k < U; ++k) {
    vec_t out;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = activate<T, ACT>(v[k][e] * rstd * w[e] + b[e]);
    put(y, first + (uint32_t)k * step, out);
  }
}

template <typename T, int LANES, int V, int U, int ACT>
__global__ __launch_bounds__(LANES, 4) void image_backward(Args<T> p) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ T lds[2][LANES / 64];
  __shared__ T each[2][LANES * V];            // [row][channel]: the lanes' sums
  const Image<T, V> t(p);
  if (!t.there) return;
  const int c0 = t.g * p.per, spatial = (int)p.spatial;
  vec_t h[U], d[U];                            // xhat and dz
  {
    const __amdgpu_buffer_rsrc_t x = rows_of(p.x + t.n * p.x_n + c0, p.spatial, p.x_s, p.per);
    const __amdgpu_buffer_rsrc_t dy = rows_of(p.dy + t.n * p.dy_n + c0, p.spatial, p.dy_s, p.per);
    const uint32_t x0 = t.first(p.x_s), xs = (uint32_t)(p.rows_at_once * p.x_s * (int64_t)sizeof(T));
    const uint32_t d0 = t.first(p.dy_s), ds = (uint32_t)(p.rows_at_once * p.dy_s * (int64_t)sizeof(T));
#pragma unroll
    for (int k = 0; k < U; ++k) {
      h[k] = get<vec_t>(x, x0 + (uint32_t)k * xs);
      d[k] = get<vec_t>(dy, d0 + (uint32_t)k * ds);
    }
  }
  const T mean = p.mean[t.n * p.groups + t.g], rstd = p.rstd[t.n * p.groups + t.g];
  constexpr int H = V == 1 ? 2 : 1;            // two short sums in place of one of 48 rows
  T w[V], b[V], dw[H * V], db[H * V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    w[e] = p.weight ? p.weight[c0 + t.c + e] : (T)1;
    b[e] = p.bias ? p.bias[c0 + t.c + e] : (T)0;
  }
#pragma unroll
  for (int e = 0; e < H * V; ++e) dw[e] = db[e] = (T)0;
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const bool is = t.live && t.row + k * p.rows_at_once < spatial;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      h[k][e] = (h[k][e] - mean) * rstd;
      d[k][e] = is ? through<T, ACT>(d[k][e], h[k][e] * w[e] + b[e]) : (T)0;
      dw[e + k % H] += is ? d[k][e] * h[k][e] : (T)0;
      db[e + k % H] += d[k][e];
    }
  }
  if constexpr (H == 2) { dw[0] += dw[1]; db[0] += db[1]; }
  T s1 = (T)0, s2 = (T)0;
#pragma unroll
  for (int e = 0; e < V; ++e) { s1 += db[e] * w[e]; s2 += dw[e] * w[e]; }
  if (p.share && t.live)
#pragma unroll
    for (int e = 0; e < V; ++e) {
      each[0][t.row * p.per + t.c + e] = dw[e];
      each[1][t.row * p.per + t.c + e] = db[e];
    }
  image_sums(s1, s2, lds);                     // (its barriers stand between `each` being written and read)
  const T count = (T)((T)p.spatial * (T)p.per);
  s1 /= count;
  s2 /= count;
  const __amdgpu_buffer_rsrc_t dx = rows_of(p.y + t.n * p.y_n + c0, p.spatial, p.y_s, p.per);
  const uint32_t first = t.first(p.y_s), step = (uint32_t)(p.rows_at_once * p.y_s * (int64_t)sizeof(T));
#pragma unroll
  for (int k = 0; k < U; ++k) {
    vec_t out;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = rstd * (d[k][e] * w[e] - s1 - h[k][e] * s2);
    put(dx, first + (uint32_t)k * step, out);
  }
  if (!p.share) return;
  // a wavefront per sum
  for (int i = (int)threadIdx.x >> 6; i < 2 * p.per; i += LANES / 64) {
    const int c = i >> 1, lane = (int)threadIdx.x & 63;
    T sum = (T)0;
    for (int r = lane; r < p.rows_at_once; r += 64) sum += each[i & 1][r * p.per + c];
    for (int dd = 32; dd >= 1; dd >>= 1) sum += __shfl_xor(sum, dd, 64);
    if (lane == 0) p.share[(t.n * p.channels + c0 + c) * 2 + (i & 1)] = sum;
  }
}

// Where a lane of the slab kernels stands: its sample, slab, first channel and first row.
struct Place { int64_t n; int slab, c, row0; bool live; };
template <typename T, int V> __device__ __forceinline__ Place place(const Args<T>& p, unsigned id) {
  uint32_t tile, slab;
  const uint32_t rest = p.tiles_div.divmod(id, tile);
  Place w;
  w.n = p.slabs_div.divmod(rest, slab);
  w.slab = (int)slab;
  w.row0 = (int)threadIdx.x / p.lanes;
  w.c = ((int)tile * 256 + (int)threadIdx.x - w.row0 * p.lanes) * V;
  w.live = w.row0 < p.rows_at_once && w.c < p.channels;
  return w;
}

// Rows of a slab.
template <typename T> __device__ __forceinline__ int64_t rows_of_slab(const Args<T>& p, int64_t slab) {
  const int64_t left = p.spatial - slab * p.rows_per_slab;
  return left < p.rows_per_slab ? left : p.rows_per_slab;
}

// Per slab and channel: the mean of x and its squared deviations from it; BWD: the sums of dz * xhat and dz.
// Forwards a lane takes its rows in runs of 64: the sums of d = x - m and of d * d, m being its mean so far (of the first run: its
// first element), then m <- m + sum d / n and squares <- squares + sum d^2 - (sum d)^2 / n with n the rows up to there. The subtraction
// loses at most a factor of 64 in the first run, and of 2 later, however far the first element lies from the others; for double
// images of 40000 elements around 1000 behind a first 0, sums about that 0 were off by 10^-11.
template <typename T, int V, bool BWD, int ACT>
__global__ __launch_bounds__(256) void slab_sums(Args<T> p) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ double lds[256 * V * 2];
  const Place w = place<T, V>(p, blockIdx.x);
  double a[V], b[V], m[V], sq[V];
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = b[e] = m[e] = sq[e] = 0.0;
  const int64_t lo = (int64_t)w.slab * p.rows_per_slab;
  const int64_t hi = lo + rows_of_slab(p, w.slab);
  if (w.live) {
    T mean[V], rstd[V], wt[V], bs[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (BWD) {
        const int g = (int)p.per_div.div((uint32_t)(w.c + e));
        wt[e] = p.weight ? p.weight[w.c + e] : (T)1;
        bs[e] = p.bias ? p.bias[w.c + e] : (T)0;
        mean[e] = p.mean[w.n * p.groups + g];
        rstd[e] = p.rstd[w.n * p.groups + g];
      }
    }
    const T* x = p.x + w.n * p.x_n + w.c;
    const T* dy = BWD ? p.dy + w.n * p.dy_n + w.c : nullptr;
    constexpr int R = 4;                         // rows on their way at once
    int64_t s = lo + w.row0, taken = 0, seen = 0;   // forwards: rows in the sums, and in the mean
    if constexpr (!BWD) {
      if (s < hi) {
        const vec_t first = *(const vec_t*)(x + s * p.x_s);
#pragma unroll
        for (int e = 0; e < V; ++e) m[e] = (double)first[e];
      }
    }
    auto settle = [&]() {
      seen += taken;
      taken = 0;
      const double share = 1.0 / (double)seen;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double t = a[e] * share;
        sq[e] += b[e] - a[e] * t;
        m[e] += t;
        a[e] = b[e] = 0.0;
      }
    };
    for (; s + (R - 1) * p.rows_at_once < hi; s += R * p.rows_at_once) {
      vec_t xv[R], dv[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        xv[r] = *(const vec_t*)(x + (s + r * p.rows_at_once) * p.x_s);
        if constexpr (BWD) dv[r] = *(const vec_t*)(dy + (s + r * p.rows_at_once) * p.dy_s);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (BWD) {                     // four rows in T, then on in double
          T ha = (T)0, hb = (T)0;
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const T h = (xv[r][e] - mean[e]) * rstd[e];
            const T dz = through<T, ACT>(dv[r][e], h * wt[e] + bs[e]);
            ha += dz * h;
            hb += dz;
          }
          a[e] += (double)ha;
          b[e] += (double)hb;
        } else {
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const double d = (double)xv[r][e] - m[e];
            a[e] += d;
            b[e] += d * d;
          }
        }
      }
      if constexpr (!BWD) {
        taken += R;
        if (taken == 64) settle();
      }
    }
    for (; s < hi; s += p.rows_at_once) {
      const vec_t xv = *(const vec_t*)(x + s * p.x_s);
      vec_t dv;
      if constexpr (BWD) dv = *(const vec_t*)(dy + s * p.dy_s);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if constexpr (BWD) {
          const T h = (xv[e] - mean[e]) * rstd[e];
          const T dz = through<T, ACT>(dv[e], h * wt[e] + bs[e]);
          a[e] += (double)(dz * h);
          b[e] += (double)dz;
        } else {
          const double d = (double)xv[e] - m[e];
          a[e] += d;
          b[e] += d * d;
        }
      }
      if constexpr (!BWD) ++taken;
    }
    if constexpr (!BWD) {
      if (taken) settle();
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    lds[(threadIdx.x * V + e) * 2] = BWD ? a[e] : m[e];
    lds[(threadIdx.x * V + e) * 2 + 1] = BWD ? b[e] : sq[e];
  }
  __syncthreads();
  if (!w.live || w.row0 != 0) return;
  double* out = p.part + ((w.n * p.slabs + w.slab) * (int64_t)p.channels + w.c) * 2;
  const int64_t rows = hi - lo;
  const int lanes = rows < p.rows_at_once ? (int)rows : p.rows_at_once;   // lanes that have rows of this slab
#pragma unroll
  for (int e = 0; e < V; ++e) {
    auto at = [&](int r) { return (threadIdx.x + r * p.lanes) * V + e; };
    if constexpr (BWD) {
      for (int r = 1; r < p.rows_at_once; ++r) {
        a[e] += lds[at(r) * 2];
        b[e] += lds[at(r) * 2 + 1];
      }
      out[2 * e] = a[e];
      out[2 * e + 1] = b[e];
    } else {
      // the lanes' means and squares: the first (rows % rows_at_once) lanes have a row more than the others
      const double few = (double)(rows / p.rows_at_once);
      const int more = (int)(rows % p.rows_at_once);
      double shift = 0.0;
      for (int r = 1; r < lanes; ++r) shift += (few + (r < more ? 1.0 : 0.0)) * (lds[at(r) * 2] - m[e]);
      const double all = m[e] + shift / (double)rows;
      double squares = 0.0;
      for (int r = 0; r < lanes; ++r) {
        const double d = lds[at(r) * 2] - all;
        squares += lds[at(r) * 2 + 1] + (few + (r < more ? 1.0 : 0.0)) * (d * d);
      }
      out[2 * e] = all;
      out[2 * e + 1] = squares;
    }
  }
}

// The sum of `v` over the workgroup of 256, in a fixed order, the same in every lane.
__device__ __forceinline__ Vec<double, 2>::type fold_256(Vec<double, 2>::type v, Vec<double, 2>::type (&lds)[256]) {
  __syncthreads();
  lds[threadIdx.x] = v;
  __syncthreads();
  for (int d = 128; d >= 1; d >>= 1) {
    if ((int)threadIdx.x < d) lds[threadIdx.x] += lds[threadIdx.x + d];
    __syncthreads();
  }
  return lds[0];
}

// The slabs of one group, in a fixed order. Forwards mean and rstd from the slabs' means and squares, in two passes over them (the
// second one's reading is still in the die's L2); BWD the two averages of the backward pass and, where they are wanted, each channel's
// sums over the sample. A lane stays with one channel (of up to 256 at a time) and takes every so many-th slab.
template <typename T, bool BWD>
__global__ __launch_bounds__(256) void group_fold(Args<T> p) {
  typedef Vec<double, 2>::type pair_t;
  __shared__ pair_t lds[256];
  uint32_t g;
  const int64_t n = p.groups_div.divmod(blockIdx.x, g);
  const pair_t* part = (const pair_t*)p.part + n * p.slabs * (int64_t)p.channels + (int64_t)g * p.per;
  const int wide = p.per < 256 ? p.per : 256, rows = 256 / wide;
  const int k = (int)threadIdx.x / wide, cl = (int)threadIdx.x - k * wide;
  // take(pair, slab) for every slab of the lane's row in channel c
  auto each = [&](int c, auto take) {
    int i = k;
    for (; i + 7 * rows < p.slabs; i += 8 * rows) {
      pair_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = part[(int64_t)(i + u * rows) * p.channels + c];
#pragma unroll
      for (int u = 0; u < 8; ++u) take(v[u], i + u * rows);
    }
    for (; i < p.slabs; i += rows) take(part[(int64_t)i * p.channels + c], i);
  };
  const double count = (double)p.spatial * (double)p.per;
  const int64_t at = n * p.groups + g;
  if constexpr (BWD) {
    pair_t all = (pair_t)(0.0);                            // lanes of row 0: their channels' sums
    for (int c0 = 0; c0 < p.per; c0 += wide) {
      const int c = c0 + cl;
      const bool live = k < rows && c < p.per;
      pair_t s = (pair_t)(0.0);
      if (live) each(c, [&](pair_t v, int) { s += v; });
      __syncthreads();
      lds[threadIdx.x] = s;
      __syncthreads();
      if (live && k == 0) {
        for (int r = 1; r < rows; ++r) s += lds[threadIdx.x + r * wide];
        if (p.chan) ((pair_t*)p.chan)[n * p.channels + (int64_t)g * p.per + c] = s;
        all += s * (p.weight ? (double)p.weight[g * p.per + c] : 1.0);
      }
    }
    all = fold_256(all, lds);
    if (threadIdx.x) return;
    p.coef[2 * at] = (T)(all[1] / count);
    p.coef[2 * at + 1] = (T)(all[0] / count);
  } else {
    const double pivot = part[0][0];
    pair_t s = (pair_t)(0.0);
    for (int c = cl; c < p.per && k < rows; c += wide) each(c, [&](pair_t v, int i) { s[0] += (double)rows_of_slab(p, i) * (v[0] - pivot); });
    const double mean = pivot + fold_256(s, lds)[0] / count;
    s = (pair_t)(0.0);
    for (int c = cl; c < p.per && k < rows; c += wide)
      each(c, [&](pair_t v, int i) { s[1] += v[1] + (double)rows_of_slab(p, i) * ((v[0] - mean) * (v[0] - mean)); });
    const double var = fold_256(s, lds)[1] / count;
    if (threadIdx.x) return;
    p.mean[at] = (T)mean;
    p.rstd[at] = (T)(1.0 / sqrt(var + (double)p.eps));
  }
}

// dweight and dbias of 8 channels: 8 lanes side by side, 32 of them over the parts, folded through LDS. Part i (slot, row) of
// channel c (group, channel of it) lies at ((slot * groups + group) * rows + row) * per + channel; rows = 1: at i * channels + c.
template <int DEPTH, typename T, typename P>
__device__ __forceinline__ void fold_channels(const Args<T>& p, const P* part, int64_t slots, int rows, bool add, int block) {
  typedef typename Vec<P, 2>::type pair_t;
  __shared__ double lds[256][2];
  const int c = block * 8 + ((int)threadIdx.x & 7), k = (int)threadIdx.x >> 3;
  double a = 0.0, b = 0.0;
  if (c < p.channels) {
    uint32_t cg;
    const uint32_t g = p.per_div.divmod((uint32_t)c, cg);
    const pair_t* at = (const pair_t*)part + (int64_t)g * rows * p.per + cg;
    const int64_t pitch = (int64_t)p.channels * rows, parts = slots * rows;
    auto where = [&](int64_t i) { const int64_t slot = rows == 1 ? i : i / rows; return slot * pitch + (i - slot * rows) * p.per; };
    int64_t i = k;
    for (; i + (DEPTH - 1) * 32 < parts; i += DEPTH * 32) {
      pair_t v[DEPTH];
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) v[u] = at[where(i + u * 32)];
#pragma unroll
      for (int u = 0; u < DEPTH; ++u) { a += (double)v[u][0]; b += (double)v[u][1]; }
    }
    for (; i < parts; i += 32) { const pair_t v = at[where(i)]; a += (double)v[0]; b += (double)v[1]; }
  }
  lds[threadIdx.x][0] = a;
  lds[threadIdx.x][1] = b;
  __syncthreads();
  if (k != 0 || c >= p.channels) return;
#pragma unroll 4                     // (all at once is 132 registers, for every wavefront of the second pass)
  for (int r = 1; r < 32; ++r) { a += lds[threadIdx.x + 8 * r][0]; b += lds[threadIdx.x + 8 * r][1]; }
  if (p.dweight) p.dweight[c] = (T)(add ? (double)p.dweight[c] + a : a);
  if (p.dbias) p.dbias[c] = (T)(add ? (double)p.dbias[c] + b : b);
}

template <typename T, typename P>
__global__ __launch_bounds__(256) void channel_fold(Args<T> p, const P* part, int64_t slots, int rows, bool add) {
  fold_channels<8>(p, part, slots, rows, add, (int)blockIdx.x);
}

// Sums over `each` samples at a time of [samples, columns] (a lane stays with a column), in a fixed order.
template <typename P>
__global__ __launch_bounds__(256) void sample_sums(const P* part, double* out, int64_t samples, int64_t each, int columns) {
  const int c = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (c >= columns) return;
  const int64_t lo = (int64_t)blockIdx.y * each, hi = lo + each < samples ? lo + each : samples;
  double sum = 0.0;
  int64_t i = lo;
  for (; i + 7 < hi; i += 8) {
    P v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = part[(i + u) * columns + c];
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += (double)v[u];
  }
  for (; i < hi; ++i) sum += (double)part[i * columns + c];
  out[(int64_t)blockIdx.y * columns + c] = sum;
}

// Second pass over the slabs: y from mean and rstd, or (BWD) dx from the averages too.
template <typename T, int V, bool BWD, int ACT, bool NT>
__global__ __launch_bounds__(256) void slab_apply(Args<T> p) {
  typedef typename Vec<T, V>::type vec_t;
  if constexpr (BWD) {
    if (blockIdx.x < (unsigned)p.folds) {                  // uniform
      fold_channels<4>(p, (const double*)p.chan, p.nc, 1, p.n0 > 0, (int)blockIdx.x);
      return;
    }
  }
  const Place w = place<T, V>(p, blockIdx.x - (BWD ? (unsigned)p.folds : 0u));
  if (!w.live) return;
  T mean[V], rstd[V], wt[V], bs[V], c1[V], c2[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int64_t g = w.n * p.groups + p.per_div.div((uint32_t)(w.c + e));
    mean[e] = p.mean[g];
    rstd[e] = p.rstd[g];
    wt[e] = p.weight ? p.weight[w.c + e] : (T)1;
    bs[e] = p.bias ? p.bias[w.c + e] : (T)0;
    if constexpr (BWD) { c1[e] = p.coef[2 * g]; c2[e] = p.coef[2 * g + 1]; }
  }
  const int64_t lo = (int64_t)w.slab * p.rows_per_slab;
  const int64_t hi = lo + p.rows_per_slab < p.spatial ? lo + p.rows_per_slab : p.spatial;
#pragma unroll 4
  for (int64_t s = lo + w.row0; s < hi; s += p.rows_at_once) {
    const vec_t xv = fetch<NT>((const vec_t*)(p.x + w.n * p.x_n + s * p.x_s + w.c));
    vec_t out;
    if constexpr (BWD) {
      const vec_t dv = fetch<NT>((const vec_t*)(p.dy + w.n * p.dy_n + s * p.dy_s + w.c));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const T h = (xv[e] - mean[e]) * rstd[e];
        const T dz = through<T, ACT>(dv[e], h * wt[e] + bs[e]);
        out[e] = rstd[e] * (dz * wt[e] - c1[e] - h * c2[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) out[e] = activate<T, ACT>((xv[e] - mean[e]) * rstd[e] * wt[e] + bs[e]);
    }
    *(vec_t*)(p.y + w.n * p.y_n + s * p.y_s + w.c) = out;
  }
}

template <typename T>
__global__ __launch_bounds__(256) void clear(T* a, T* b, int n) {
  const int i = (int)blockIdx.x * 256 + (int)threadIdx.x;
  if (i >= n) return;
  if (a) a[i] = (T)0;
  if (b) b[i] = (T)0;
}

// How a team covers a group of `units` vectors: the narrowest team that holds four vectors a lane, or a workgroup with up to
// eight; 0 when it does not fit.
static int team_lanes(int64_t units) {
  for (int l = 8; l <= 64; l *= 2)
    if (units <= (int64_t)l * 4) return l;
  return units <= 256 * kUnits ? 256 : 0;
}

template <typename T> static void set_slabs(Args<T>& p, int V, int64_t rows, int64_t samples) {
  const int cv = p.channels / V;
  p.tiles = (cv + 255) / 256;
  p.lanes = cv < 256 ? cv : 256;
  p.rows_at_once = 256 / p.lanes;
  // a few workgroups for every CU, of at least eight rows for each lane
  int64_t slabs = ((int64_t)num_cus() * 4 + samples * p.tiles - 1) / (samples * p.tiles);
  const int64_t most = (rows + p.rows_at_once * 8 - 1) / (p.rows_at_once * 8);
  if (slabs > most) slabs = most;
  if (slabs < 1) slabs = 1;
  p.rows_per_slab = (rows + slabs - 1) / slabs;
  p.slabs = (int)((rows + p.rows_per_slab - 1) / p.rows_per_slab);
  p.tiles_div = FastDiv((uint32_t)p.tiles);
  p.slabs_div = FastDiv((uint32_t)p.slabs);
}

// dweight and dbias from every sample's sums per channel, [samples, channels, 2]. Many samples are added up in 128 runs first:
// channel_fold has a workgroup for 8 channels, and no more of them ([8192, 16, 8, 16] in 1 group, backwards 79 -> 63 us).
template <typename T, typename P>
static int fold_samples(const Args<T>& p, const P* part, int64_t samples, bool add) {
  const dim3 grid((unsigned)((p.channels + 7) / 8)), block(256);
  if (samples <= 512) {
    hipLaunchKernelGGL((channel_fold<T, P>), grid, block, 0, stream(), p, part, samples, 1, add);
    return check_launch("channel_fold");
  }
  const int64_t each = (samples + 127) / 128, runs = (samples + each - 1) / each;
  const int columns = 2 * p.channels;
  Scratch sums;
  AM_TRY(sums.take((size_t)runs * columns * sizeof(double)));
  hipLaunchKernelGGL((sample_sums<P>), dim3((unsigned)((columns + 255) / 256), (unsigned)runs), block, 0, stream(), part, (double*)sums.p, samples, each, columns);
  AM_TRY(check_launch("sample_sums"));
  hipLaunchKernelGGL((channel_fold<T, double>), grid, block, 0, stream(), p, (const double*)sums.p, runs, 1, add);
  return check_launch("channel_fold");
}

#define AM_GN_LAUNCH(KERNEL, V_, GRID, ...)                                                                         \
  do {                                                                                                              \
    const dim3 grid_((unsigned)(GRID)), block_(256);                                                                \
    if (V_ > 1) hipLaunchKernelGGL((KERNEL<T, W, __VA_ARGS__>), grid_, block_, 0, stream(), p);                      \
    else hipLaunchKernelGGL((KERNEL<T, 1, __VA_ARGS__>), grid_, block_, 0, stream(), p);                             \
  } while (0)

constexpr size_t kMostScratch = (size_t)256 << 20;
constexpr int64_t kMostThreads = ((int64_t)1 << 32) - 1;     // of a launch

// Samples of a slab launch: as many as the scratch memory and a launch hold (beside the workgroups that fold up to 2^24 channels).
template <typename T> static int64_t samples_at_once(const Args<T>& p, size_t per_sample) {
  const int64_t wgs = (int64_t)p.slabs * p.tiles > p.groups ? (int64_t)p.slabs * p.tiles : p.groups;
  int64_t nc = (int64_t)(kMostScratch / per_sample);
  const int64_t launch = (kMostThreads / 256 - ((int64_t)1 << 21)) / wgs;
  if (nc > launch) nc = launch;
  if (nc < 1) nc = 1;
  return nc < p.batch ? nc : p.batch;
}

template <typename T> static bool fits(const void* base, int64_t sn, int64_t ss, int64_t batch, int64_t spatial) {
  constexpr int64_t W = 16 / (int64_t)sizeof(T);
  return (uintptr_t)base % 16 == 0 && (sn % W == 0 || batch == 1) && (ss % W == 0 || spatial == 1);
}

template <typename T>
static int check_args(const char* fn, int64_t batch, int64_t spatial, int64_t channels, int64_t groups, int activation) {
  if (activation < AM_ACT_NONE || activation > AM_ACT_SILU) return fail(AM_E_ARG, "%s: unknown activation %d", fn, activation);
  if (batch < 0 || spatial < 0 || channels < 0) return fail(AM_E_SHAPE, "%s: negative extent", fn);
  if (groups < 1 || channels % groups) return fail(AM_E_SHAPE, "%s: %lld channels in %lld groups", fn, (long long)channels, (long long)groups);
  if (channels >= ((int64_t)1 << 24) || spatial >= ((int64_t)1 << 40) || batch >= ((int64_t)1 << 31)) return fail(AM_E_SHAPE, "%s: extent too large", fn);
  return AM_OK;
}

// Whether x is larger than the caches keep and not read again: who asks for the statistics has a backward pass to come
// ([16, 64, 64, 320] forwards and backwards 158 us with x read past the caches, 141 without).
template <bool BWD, typename T> static bool last_reading(const Args<T>& p) {
  return (BWD || !p.mean) && (double)p.batch * (double)p.spatial * p.channels * sizeof(T) > nt_threshold_bytes();
}

template <typename T, int V, int U, bool WIDE, int ACT, bool BWD>
static void launch_team(const Args<T>& p, int lanes, int units, int64_t slots, int64_t wgs) {
  const dim3 grid((unsigned)wgs), block(256);
  const bool nt = V > 1 && last_reading<BWD>(p);
  if constexpr (BWD) {
    if (nt) hipLaunchKernelGGL((team_backward<T, V, U, WIDE, ACT, (V > 1)>), grid, block, 0, stream(), p, lanes, units, slots);
    else hipLaunchKernelGGL((team_backward<T, V, U, WIDE, ACT, false>), grid, block, 0, stream(), p, lanes, units, slots);
  } else {
    if (nt) hipLaunchKernelGGL((team_forward<T, V, U, WIDE, ACT, (V > 1)>), grid, block, 0, stream(), p, lanes, units, slots);
    else hipLaunchKernelGGL((team_forward<T, V, U, WIDE, ACT, false>), grid, block, 0, stream(), p, lanes, units, slots);
  }
}

template <typename T, int V, int ACT, bool BWD>
static int team_pass(Args<T> p, int lanes, int units) {
  // Samples per team: as many as leave eight workgroups for every CU (backwards two, as the shares of the parameters'
  // gradients have to be written and read again: [16384, 2048] in 16 groups 88 us, against 96 with one and 100 with four), and at most 64: a lane's shares are sums of that many
  // terms in the result's type, 64 roundings at most (in double they would take twice the registers, which hold the sample as well),
  // and go on in double in `channel_fold`. They keep every row of a sample, with few samples a team up to twice x in memory.
  const int64_t at_once = 256 / lanes;
  int64_t slots = (int64_t)num_cus() * (BWD ? 2 : 8) * at_once / p.groups;
  if (slots < (p.batch + 63) / 64) slots = (p.batch + 63) / 64;
  if (slots < 1) slots = 1;
  if (slots > p.batch) slots = p.batch;
  const int64_t each = (p.batch + slots - 1) / slots;
  slots = (p.batch + each - 1) / each;
  const int64_t wgs = (slots * p.groups + at_once - 1) / at_once;
  if (wgs > kMostThreads / 256) return fail(AM_E_SHAPE, "group norm: too many groups for one launch");
  const int64_t rows = lanes == 256 ? 1 : p.spatial;      // of a slot's shares
  Scratch share;
  if (BWD && (p.dweight || p.dbias)) {
    AM_TRY(share.take((size_t)slots * p.channels * (size_t)rows * 2 * sizeof(T)));
    p.share = (T*)share.p;
  }
  const int per_lane = (units + lanes - 1) / lanes;
  if (lanes == 256) {
    if (per_lane <= 2) launch_team<T, V, 2, true, ACT, BWD>(p, lanes, units, slots, wgs);
    else if (per_lane <= 4) launch_team<T, V, 4, true, ACT, BWD>(p, lanes, units, slots, wgs);
    else launch_team<T, V, 8, true, ACT, BWD>(p, lanes, units, slots, wgs);
  } else {
    if (per_lane == 1) launch_team<T, V, 1, false, ACT, BWD>(p, lanes, units, slots, wgs);
    else if (per_lane == 2) launch_team<T, V, 2, false, ACT, BWD>(p, lanes, units, slots, wgs);
    else launch_team<T, V, 4, false, ACT, BWD>(p, lanes, units, slots, wgs);
  }
  AM_TRY(check_launch("group norm of teams"));
  if (p.share) {
    hipLaunchKernelGGL((channel_fold<T, T>), dim3((unsigned)((p.channels + 7) / 8)), dim3(256), 0, stream(), p, (const T*)p.share, slots, (int)rows, false);
    AM_TRY(check_launch("channel_fold"));
  }
  return AM_OK;
}

// The team's way, if the groups fit it: AM_OK + taken.
template <typename T, int ACT, bool BWD>
static int try_teams(Args<T>& p, bool aligned, bool& taken) {
  constexpr int W = 16 / (int)sizeof(T);
  const int V = aligned && p.per % W == 0 ? W : 1;
  const int64_t upr = p.per / V;
  const int lanes = p.spatial <= 256 * kUnits ? team_lanes(p.spatial * upr) : 0;
  taken = lanes > 0;
  if (!taken) return AM_OK;
  p.units_div = FastDiv((uint32_t)upr);
  const int units = (int)(p.spatial * upr);
  return V > 1 ? team_pass<T, W, ACT, BWD>(p, lanes, units) : team_pass<T, 1, ACT, BWD>(p, lanes, units);
}

// The image's way, where a workgroup's registers hold a group.
template <typename T, int LANES, int V, int U, int ACT, bool BWD> static void launch_image(const Args<T>& p) {
  const dim3 grid((unsigned)((p.batch * p.groups + 7) / 8 * 8)), block(LANES);
  if constexpr (BWD) hipLaunchKernelGGL((image_backward<T, LANES, V, U, ACT>), grid, block, 0, stream(), p);
  else hipLaunchKernelGGL((image_forward<T, LANES, V, U, ACT>), grid, block, 0, stream(), p);
}

template <typename T, int V, int ACT, bool BWD>
static int image_pass(Args<T> p, int lanes) {
  constexpr int U = kImageHeld<T> / V;
  Scratch share;
  if (BWD && (p.dweight || p.dbias)) {
    AM_TRY(share.take((size_t)p.batch * p.channels * 2 * sizeof(T)));
    p.share = (T*)share.p;
  }
  const int64_t most = (kMostThreads / lanes - 8) / p.groups;    // samples of a launch
  for (int64_t n = 0; n < p.batch; n += most) {
    Args<T> q = p;
    q.batch = p.batch - n < most ? p.batch - n : most;
    q.x += n * p.x_n;
    q.y += n * p.y_n;
    if (BWD) q.dy += n * p.dy_n;
    if (p.mean) { q.mean += n * p.groups; q.rstd += n * p.groups; }
    if (p.share) q.share += n * p.channels * 2;
    if (lanes == 256 && p.spatial <= (int64_t)p.rows_at_once * (U / 2)) launch_image<T, 256, V, U / 2, ACT, BWD>(q);
    else if (lanes == 256) launch_image<T, 256, V, U, ACT, BWD>(q);
    else if (lanes == 512) launch_image<T, 512, V, U, ACT, BWD>(q);
    else launch_image<T, 1024, V, U, ACT, BWD>(q);
    AM_TRY(check_launch("group norm of images"));
  }
  return p.share ? fold_samples<T, T>(p, p.share, p.batch, false) : AM_OK;
}

template <typename T, int ACT, bool BWD>
static int try_images(Args<T>& p, bool aligned, bool& taken) {
  // us forwards + backwards, images against what else takes the shape.
  //  - Few rows: the teams, whose lanes hold what they need and no more ([64, 8, 8, 1024] in 32 groups 13 + 30 against 10 + 17 in
  //    teams). From 128 rows on the images: [16, 45, 45, 128] in 32 15 + 23 against 34 + 64 in teams, [512, 16, 16, 256] in 32
  //    82 + 117 against 159 + 267, [256, 16, 16, 512] in 128 128 + 174 against 221 + 500 (backwards the teams keep shares of
  //    dweight for every row); only small ones lose a little, [64, 16, 16, 128] in 32 12 + 18 against 9 + 103.
  //  - A row of a group is a short run of memory, and a cache line that several groups share is fetched for each of them unless
  //    the die's L2 still has it. From 48 bytes on that is no loss: [16, 56, 56, 384] in 32 groups 49 + 78 against 49 + 88 in
  //    slabs, with 64 bytes ([32, 48, 48, 256] in 16) 43 + 63 against 47 + 81, with 256 ([16, 24, 24, 1024] in 16) 19 + 30 against
  //    36 + 48. From 16 bytes on it is none against slabs while the device's last cache holds the tensors: 40 bytes of 42 MB
  //    25 + 41 against 33 + 48, of 63 MB 51 + 79 against 44 + 73; 16 bytes of 17 MB 16 + 25 against 19 + 29; 12 bytes of 14 MB
  //    24 + 36 against 20 + 29.
  taken = false;
  constexpr int W = 16 / (int)sizeof(T);
  const int run = p.per * (int)sizeof(T);
  if (p.spatial < 128 || run < 16) return AM_OK;
  const bool slabs = p.spatial * (p.per / (aligned && p.per % W == 0 ? W : 1)) > 256 * kUnits;
  if (slabs && run < 48 && (double)p.batch * (double)p.spatial * p.channels * sizeof(T) > 48e6) return AM_OK;
  int V = 16 / (int)sizeof(T);
  // rows one behind the other, and all that the lanes may count up to within 2^31 bytes
  constexpr int64_t most = ((int64_t)1 << 31) / ((kImageHeld<T> + 1) * kImage * (int)sizeof(T));
  auto holds = [&](const T* base, int64_t sn, int64_t ss) {
    while (V > 1 && (p.per % V || (uintptr_t)base % (V * sizeof(T)) || sn % V || ss % V)) V /= 2;
    return (ss >= p.per || p.spatial == 1) && ss >= 0 && ss < most;
  };
  if (!holds(p.x, p.x_n, p.x_s) || !holds(p.y, p.y_n, p.y_s)) return AM_OK;
  if (BWD && !holds(p.dy, p.dy_n, p.dy_s)) return AM_OK;
  // The fewest lanes that hold a group, so that several workgroups share a CU and one reads while another writes.
  const int64_t upr = p.per / V;
  int lanes = 256;
  while (lanes <= kImage && (upr > lanes || (p.spatial + lanes / upr - 1) / (lanes / upr) * V > kImageHeld<T>)) lanes *= 2;
  if (lanes > kImage || p.groups > kMostThreads / lanes - 8) return AM_OK;
  taken = true;
  p.units_div = FastDiv((uint32_t)upr);
  p.rows_at_once = (int)(lanes / upr);
  if constexpr (sizeof(T) == 4) {
    if (V == 4) return image_pass<T, 4, ACT, BWD>(p, lanes);
  }
  if (V == 2) return image_pass<T, 2, ACT, BWD>(p, lanes);
  return image_pass<T, 1, ACT, BWD>(p, lanes);
}

template <typename T, int ACT>
static int forward(Args<T> p) {
  constexpr int W = 16 / (int)sizeof(T);
  const bool aligned = fits<T>(p.x, p.x_n, p.x_s, p.batch, p.spatial) && fits<T>(p.y, p.y_n, p.y_s, p.batch, p.spatial);
  bool taken;
  AM_TRY((try_images<T, ACT, false>(p, aligned, taken)));
  if (taken) return AM_OK;
  AM_TRY((try_teams<T, ACT, false>(p, aligned, taken)));
  if (taken) return AM_OK;
  const int V = aligned && p.channels % W == 0 ? W : 1;
  const Args<T> all = p;
  Scratch stats;
  if (!all.mean) {
    AM_TRY(stats.take((size_t)p.batch * p.groups * 2 * sizeof(T)));
    p.mean = (T*)stats.p;
    p.rstd = p.mean + p.batch * p.groups;
  }
  T* const mean = p.mean;
  T* const rstd = p.rstd;
  set_slabs(p, V, p.spatial, p.batch);
  const size_t per_sample = (size_t)p.slabs * p.channels * 2 * sizeof(double);
  const int64_t nc = samples_at_once(p, per_sample);
  Scratch part;
  AM_TRY(part.take(per_sample * (size_t)nc));
  p.part = (double*)part.p;
  for (int64_t n = 0; n < all.batch; n += nc) {
    p.nc = all.batch - n < nc ? all.batch - n : nc;
    p.x = all.x + n * p.x_n;
    p.y = all.y + n * p.y_n;
    p.mean = mean + n * p.groups;
    p.rstd = rstd + n * p.groups;
    const int64_t wgs = p.nc * p.slabs * p.tiles;
    AM_GN_LAUNCH(slab_sums, V, wgs, false, ACT);
    AM_TRY(check_launch("slab_sums"));
    hipLaunchKernelGGL((group_fold<T, false>), dim3((unsigned)(p.nc * p.groups)), dim3(256), 0, stream(), p);
    AM_TRY(check_launch("group_fold"));
    if (V > 1 && last_reading<false>(all)) AM_GN_LAUNCH(slab_apply, V, wgs, false, ACT, true);
    else AM_GN_LAUNCH(slab_apply, V, wgs, false, ACT, false);
    AM_TRY(check_launch("slab_apply"));
  }
  return AM_OK;
}

template <typename T, int ACT>
static int backward(Args<T> p) {
  constexpr int W = 16 / (int)sizeof(T);
  const bool params = p.dweight || p.dbias;
  if (p.batch == 0 || p.spatial == 0) {
    if (!params || p.channels == 0) return AM_OK;
    hipLaunchKernelGGL((clear<T>), dim3((unsigned)((p.channels + 255) / 256)), dim3(256), 0, stream(), p.dweight, p.dbias, p.channels);
    return check_launch("clear");
  }
  const bool aligned = fits<T>(p.x, p.x_n, p.x_s, p.batch, p.spatial) && fits<T>(p.y, p.y_n, p.y_s, p.batch, p.spatial) &&
                       fits<T>(p.dy, p.dy_n, p.dy_s, p.batch, p.spatial);
  bool taken;
  AM_TRY((try_images<T, ACT, true>(p, aligned, taken)));
  if (taken) return AM_OK;
  AM_TRY((try_teams<T, ACT, true>(p, aligned, taken)));
  if (taken) return AM_OK;
  const int V = aligned && p.channels % W == 0 ? W : 1;
  const Args<T> all = p;
  Scratch part;
  set_slabs(p, V, p.spatial, p.batch);
  const size_t per_sample = (size_t)p.slabs * p.channels * 2 * sizeof(double);
  const int64_t nc = samples_at_once(p, per_sample);
  const size_t coef_bytes = (size_t)nc * p.groups * 2 * sizeof(T);
  const size_t part_bytes = per_sample * (size_t)nc, chan_bytes = params ? (size_t)nc * p.channels * 2 * sizeof(double) : 0;
  AM_TRY(part.take(part_bytes + chan_bytes + coef_bytes));
  p.part = (double*)part.p;
  p.chan = params ? (double*)((char*)part.p + part_bytes) : nullptr;
  p.coef = (T*)((char*)part.p + part_bytes + chan_bytes);
  for (int64_t n = 0; n < all.batch; n += nc) {
    p.nc = all.batch - n < nc ? all.batch - n : nc;
    p.x = all.x + n * p.x_n;
    p.y = all.y + n * p.y_n;
    p.dy = all.dy + n * p.dy_n;
    p.mean = all.mean + n * p.groups;
    p.rstd = all.rstd + n * p.groups;
    const int64_t wgs = p.nc * p.slabs * p.tiles;
    AM_GN_LAUNCH(slab_sums, V, wgs, true, ACT);
    AM_TRY(check_launch("slab_sums"));
    hipLaunchKernelGGL((group_fold<T, true>), dim3((unsigned)(p.nc * p.groups)), dim3(256), 0, stream(), p);
    AM_TRY(check_launch("group_fold"));
    // Few samples' sums per channel are folded beside the second pass ([16, 64, 64, 320] 89.8 -> 87.3 us), many before it.
    p.n0 = n;
    p.folds = params && p.nc <= 512 ? (p.channels + 7) / 8 : 0;
    if (params && !p.folds) AM_TRY((fold_samples<T, double>(p, p.chan, p.nc, n > 0)));
    AM_GN_LAUNCH(slab_apply, V, wgs + p.folds, true, ACT, false);   // (past the caches 89.5 -> 94 us for [16, 64, 64, 320])
    AM_TRY(check_launch("slab_apply"));
  }
  return AM_OK;
}

template <typename T> static void set_common(Args<T>& p, int64_t batch, int64_t spatial, int64_t channels, int64_t groups) {
  p.batch = batch; p.spatial = spatial;
  p.channels = (int)channels; p.groups = (int)groups; p.per = (int)(channels / groups);
  p.per_div = FastDiv((uint32_t)p.per);
  p.groups_div = FastDiv((uint32_t)p.groups);
}

template <typename T>
static int run_forward(const char* fn, int64_t batch, int64_t spatial, int64_t channels, int64_t groups, T eps, int activation,
                       const T* x, int64_t x_n, int64_t x_s, const T* weight, const T* bias, T* y, int64_t y_n, int64_t y_s, T* mean, T* rstd) {
  AM_TRY(check_args<T>(fn, batch, spatial, channels, groups, activation));
  if (!(eps >= (T)0)) return fail(AM_E_ARG, "%s: eps must not be negative", fn);
  if (!mean != !rstd) return fail(AM_E_ARG, "%s: mean and rstd are kept together or not at all", fn);
  if (batch == 0 || spatial == 0 || channels == 0) return AM_OK;
  if (!x || !y) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if ((batch > 1 && y_n == 0) || (spatial > 1 && y_s == 0)) return fail(AM_E_SHAPE, "%s: the result is a broadcast view", fn);
  AM_TRY(ensure_init());
  Args<T> p = {};
  p.x = x; p.x_n = x_n; p.x_s = x_s; p.weight = weight; p.bias = bias;
  p.y = y; p.y_n = y_n; p.y_s = y_s; p.mean = mean; p.rstd = rstd; p.eps = eps;
  set_common(p, batch, spatial, channels, groups);
  switch (activation) {
    case AM_ACT_RELU: return forward<T, AM_ACT_RELU>(p);
    case AM_ACT_SILU: return forward<T, AM_ACT_SILU>(p);
    default: return forward<T, AM_ACT_NONE>(p);
  }
}

template <typename T>
static int run_backward(const char* fn, int64_t batch, int64_t spatial, int64_t channels, int64_t groups, int activation, const T* dy,
                        int64_t dy_n, int64_t dy_s, const T* x, int64_t x_n, int64_t x_s, const T* weight, const T* bias, const T* mean,
                        const T* rstd, T* dx, int64_t dx_n, int64_t dx_s, T* dweight, T* dbias) {
  AM_TRY(check_args<T>(fn, batch, spatial, channels, groups, activation));
  if (channels == 0) return AM_OK;
  if (batch && spatial) {
    if (!dy || !x || !mean || !rstd || !dx) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
    if ((batch > 1 && dx_n == 0) || (spatial > 1 && dx_s == 0)) return fail(AM_E_SHAPE, "%s: the result is a broadcast view", fn);
  }
  AM_TRY(ensure_init());
  Args<T> p = {};
  p.x = x; p.x_n = x_n; p.x_s = x_s; p.dy = dy; p.dy_n = dy_n; p.dy_s = dy_s; p.weight = weight; p.bias = bias;
  p.y = dx; p.y_n = dx_n; p.y_s = dx_s; p.mean = const_cast<T*>(mean); p.rstd = const_cast<T*>(rstd); p.dweight = dweight; p.dbias = dbias;
  set_common(p, batch, spatial, channels, groups);
  switch (activation) {
    case AM_ACT_RELU: return backward<T, AM_ACT_RELU>(p);
    case AM_ACT_SILU: return backward<T, AM_ACT_SILU>(p);
    default: return backward<T, AM_ACT_NONE>(p);
  }
}

}  // namespace gnorm
}  // namespace am

using namespace am;

#define AM_GROUP_NORM(S, T)                                                                                                          \
  extern "C" int am_hip_group_norm_##S(int64_t batch, int64_t spatial, int64_t channels, int64_t groups, T eps, int activation,      \
                                       const T* x, int64_t x_n, int64_t x_s, const T* weight, const T* bias, T* y, int64_t y_n,      \
                                       int64_t y_s, T* mean, T* rstd) {                                                              \
    return gnorm::run_forward<T>("am_hip_group_norm_" #S, batch, spatial, channels, groups, eps, activation, x, x_n, x_s, weight,    \
                                 bias, y, y_n, y_s, mean, rstd);                                                                     \
  }                                                                                                                                  \
  extern "C" int am_hip_group_norm_backward_##S(                                                                                     \
      int64_t batch, int64_t spatial, int64_t channels, int64_t groups, int activation, const T* dy, int64_t dy_n, int64_t dy_s,     \
      const T* x, int64_t x_n, int64_t x_s, const T* weight, const T* bias, const T* mean, const T* rstd, T* dx, int64_t dx_n,       \
      int64_t dx_s, T* dweight, T* dbias) {                                                                                          \
    return gnorm::run_backward<T>("am_hip_group_norm_backward_" #S, batch, spatial, channels, groups, activation, dy, dy_n, dy_s, x, \
                                  x_n, x_s, weight, bias, mean, rstd, dx, dx_n, dx_s, dweight, dbias);                               \
  }

AM_GROUP_NORM(f32, float)
AM_GROUP_NORM(f64, double)
