// Group normalisation with an activation over channels-last tensors: am_hip_group_norm_*, am_hip_group_norm_backward_*.
//
// x [batch, spatial, channels]; the channels form `groups` groups of `per`, and each (sample, group) is normalised over its
// spatial * per elements:
//     xhat = (x - mean) * rstd      z = xhat * weight[c] + bias[c]      y = act(z)
// Backwards, with dz = dy * act'(z) and averages over the same elements,
//     dx = rstd * (weight dz - avg(weight dz) - xhat * avg(weight dz xhat))
//     dweight[c] = sum dz xhat      dbias[c] = sum dz                       (over batch and spatial)
//
// Two ways through it:
//  - `team_*`: the elements of a group fit the registers of a team of lanes (8 .. 64, or a workgroup of 256). One launch,
//    x is read once, mean and squared deviations are two folds over registers.
//  - slabs: a workgroup takes a slab of rows of one sample and reads them whole, channels next to each other, whatever the
//    group's width; a lane owns V channels and keeps two sums for each. The slabs' sums per channel go to scratch memory
//    and a small kernel folds them in a fixed order, per group (mean, rstd, or the two averages of the backward pass) and,
//    backwards, per channel (dweight, dbias); then a second pass over the slabs writes the result. The sums of the forward
//    pass are of x - pivot, with the group's first element as pivot, in double: no cancellation where the mean is large
//    against the deviation.
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
  double* part;                      // [n][slab][channel][2]
  T* coef;                           // backward: [n][group][2], the two averages
  T eps;
  int64_t batch, spatial;
  int channels, groups, per;
  int64_t n0, nc;                    // samples of this launch: n0 .. n0 + nc
  int slabs; int64_t rows_per_slab;
  int tiles, lanes, rows_at_once;    // channel tiles; lanes per row of a tile; rows a workgroup reads at once
  FastDiv per_div, tiles_div, slabs_div, groups_div, units_div;
  int add;                           // backward: dweight / dbias are added to
};

__device__ __forceinline__ float dev_exp(float v) { return expf(v); }
__device__ __forceinline__ double dev_exp(double v) { return exp(v); }
__device__ __forceinline__ float dev_rsqrt(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double dev_rsqrt(double v) { return 1.0 / sqrt(v); }

template <typename T, int ACT> __device__ __forceinline__ T activate(T z) {
  if constexpr (ACT == AM_ACT_RELU) return ((T)0 >= z) ? (T)0 : z;
  else if constexpr (ACT == AM_ACT_SILU) return z / ((T)1 + dev_exp(-z));
  else return z;
}
// dy * act'(z)
template <typename T, int ACT> __device__ __forceinline__ T through(T dy, T z) {
  if constexpr (ACT == AM_ACT_RELU) return ((T)0 >= z) ? (T)0 : dy;
  else if constexpr (ACT == AM_ACT_SILU) {
    const T s = (T)1 / ((T)1 + dev_exp(-z));
    return dy * (s * ((T)1 + z * ((T)1 - s)));
  } else return dy;
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

// Unit q of a group (sample base pointers given): row q / units-per-row, channels V * (q % units-per-row) ...
template <typename T, int V, bool WIDE, int ACT>
__global__ __launch_bounds__(256) void team_forward(Args<T> p, int lanes, int units) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ T lds[4];
  const int teams = WIDE ? 1 : 256 / lanes;
  const int64_t team = (int64_t)blockIdx.x * teams + (WIDE ? 0 : (int)threadIdx.x / lanes);
  const int j0 = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (lanes - 1);
  const int step = WIDE ? 256 : lanes;
  if (!WIDE && team >= p.nc * p.groups) return;       // whole teams leave together, and teams never straddle a wavefront
  const int64_t n = team / p.groups;
  const int g = (int)(team - n * p.groups);
  const T* x = p.x + n * p.x_n + (int64_t)g * p.per;
  vec_t v[kUnits];
  uint32_t row[kUnits], col[kUnits];
  T sum = (T)0;
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int q = j0 + k * step;
    if (q < units) {
      row[k] = p.units_div.divmod((uint32_t)q, col[k]);
      v[k] = *(const vec_t*)(x + row[k] * p.x_s + col[k] * V);
    }
  }
#pragma unroll
  for (int k = 0; k < kUnits; ++k)
    if (j0 + k * step < units)
#pragma unroll
      for (int e = 0; e < V; ++e) sum += v[k][e];
  const T count = (T)((T)p.spatial * (T)p.per);
  const T mean = team_sum<T, WIDE>(sum, lanes, lds) / count;
  T sq = (T)0;
#pragma unroll
  for (int k = 0; k < kUnits; ++k)
    if (j0 + k * step < units)
#pragma unroll
      for (int e = 0; e < V; ++e) { const T d = v[k][e] - mean; sq += d * d; }
  const T rstd = dev_rsqrt(team_sum<T, WIDE>(sq, lanes, lds) / count + p.eps);
  if (j0 == 0 && p.mean) { p.mean[team] = mean; p.rstd[team] = rstd; }
  T* y = p.y + n * p.y_n + (int64_t)g * p.per;
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (j0 + k * step >= units) continue;
    const int c = g * p.per + (int)col[k] * V;
    vec_t out;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      T z = (v[k][e] - mean) * rstd;
      if (p.weight) z *= p.weight[c + e];
      if (p.bias) z += p.bias[c + e];
      out[e] = activate<T, ACT>(z);
    }
    *(vec_t*)(y + row[k] * p.y_s + col[k] * V) = out;
  }
}

template <typename T, int V, bool WIDE, int ACT>
__global__ __launch_bounds__(256) void team_backward(Args<T> p, int lanes, int units) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ T lds[4];
  const int teams = WIDE ? 1 : 256 / lanes;
  const int64_t team = (int64_t)blockIdx.x * teams + (WIDE ? 0 : (int)threadIdx.x / lanes);
  const int j0 = WIDE ? (int)threadIdx.x : (int)threadIdx.x & (lanes - 1);
  const int step = WIDE ? 256 : lanes;
  if (!WIDE && team >= p.nc * p.groups) return;
  const int64_t n = team / p.groups;
  const int g = (int)(team - n * p.groups);
  const T* x = p.x + n * p.x_n + (int64_t)g * p.per;
  const T* dy = p.dy + n * p.dy_n + (int64_t)g * p.per;
  const T mean = p.mean[team], rstd = p.rstd[team];
  vec_t h[kUnits], d[kUnits];     // xhat and weight * dz
  uint32_t row[kUnits], col[kUnits];
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    const int q = j0 + k * step;
    if (q < units) {
      row[k] = p.units_div.divmod((uint32_t)q, col[k]);
      h[k] = *(const vec_t*)(x + row[k] * p.x_s + col[k] * V);
      d[k] = *(const vec_t*)(dy + row[k] * p.dy_s + col[k] * V);
    }
  }
  T s1 = (T)0, s2 = (T)0;
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (j0 + k * step >= units) continue;
    const int c = g * p.per + (int)col[k] * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      h[k][e] = (h[k][e] - mean) * rstd;
      const T w = p.weight ? p.weight[c + e] : (T)1;
      const T z = h[k][e] * w + (p.bias ? p.bias[c + e] : (T)0);
      d[k][e] = through<T, ACT>(d[k][e], z) * w;
      s1 += d[k][e];
      s2 += d[k][e] * h[k][e];
    }
  }
  const T count = (T)((T)p.spatial * (T)p.per);
  s1 = team_sum<T, WIDE>(s1, lanes, lds) / count;
  s2 = team_sum<T, WIDE>(s2, lanes, lds) / count;
  T* dx = p.y + n * p.y_n + (int64_t)g * p.per;
#pragma unroll
  for (int k = 0; k < kUnits; ++k) {
    if (j0 + k * step >= units) continue;
    vec_t out;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = rstd * (d[k][e] - s1 - h[k][e] * s2);
    *(vec_t*)(dx + row[k] * p.y_s + col[k] * V) = out;
  }
}

// Where a lane of the slab kernels stands: its sample, slab, first channel and first row.
struct Place { int64_t n; int slab, c, row0; bool live; };
template <typename T, int V> __device__ __forceinline__ Place place(const Args<T>& p) {
  uint32_t tile, slab;
  const uint32_t rest = p.tiles_div.divmod(blockIdx.x, tile);
  Place w;
  w.n = p.slabs_div.divmod(rest, slab);
  w.slab = (int)slab;
  w.row0 = (int)threadIdx.x / p.lanes;
  w.c = ((int)tile * 256 + (int)threadIdx.x - w.row0 * p.lanes) * V;
  w.live = w.row0 < p.rows_at_once && w.c < p.channels;
  return w;
}

// Per slab and channel: the sums of x - pivot and of its square; BWD: the sums of dz and dz * xhat. FLAT (BWD): the slabs
// cut the rows of all samples together (their sums are wanted per channel only), and a row's sample is its index / spatial.
template <typename T, int V, bool BWD, bool FLAT, int ACT>
__global__ __launch_bounds__(256) void slab_sums(Args<T> p) {
  typedef typename Vec<T, V>::type vec_t;
  __shared__ double lds[256 * V * 2];
  const Place w = place<T, V>(p);
  double a[V], b[V];
#pragma unroll
  for (int e = 0; e < V; ++e) a[e] = b[e] = 0.0;
  const int64_t rows = FLAT ? p.nc * p.spatial : p.spatial;
  const int64_t lo = (int64_t)w.slab * p.rows_per_slab;
  const int64_t hi = lo + p.rows_per_slab < rows ? lo + p.rows_per_slab : rows;
  if (w.live) {
    T pivot[V], mean[V], rstd[V], wt[V], bs[V];
    int g[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
      g[e] = (int)p.per_div.div((uint32_t)(w.c + e));
      if constexpr (BWD) {
        wt[e] = p.weight ? p.weight[w.c + e] : (T)1;
        bs[e] = p.bias ? p.bias[w.c + e] : (T)0;
        if constexpr (!FLAT) { mean[e] = p.mean[w.n * p.groups + g[e]]; rstd[e] = p.rstd[w.n * p.groups + g[e]]; }
      } else {
        pivot[e] = p.x[w.n * p.x_n + (int64_t)g[e] * p.per];
      }
    }
#pragma unroll 4
    for (int64_t r = lo + w.row0; r < hi; r += p.rows_at_once) {
      int64_t n = w.n, s = r;
      if constexpr (FLAT) { n = p.spatial == 1 ? r : r / p.spatial; s = r - n * p.spatial; }
      const vec_t xv = *(const vec_t*)(p.x + n * p.x_n + s * p.x_s + w.c);
      if constexpr (BWD) {
        const vec_t dv = *(const vec_t*)(p.dy + n * p.dy_n + s * p.dy_s + w.c);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          T m, q;
          if constexpr (FLAT) { m = p.mean[n * p.groups + g[e]]; q = p.rstd[n * p.groups + g[e]]; }
          else { m = mean[e]; q = rstd[e]; }
          const T h = (xv[e] - m) * q;
          const T dz = through<T, ACT>(dv[e], h * wt[e] + bs[e]);
          a[e] += (double)dz;
          b[e] += (double)dz * (double)h;
        }
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const double d = (double)xv[e] - (double)pivot[e];
          a[e] += d;
          b[e] += d * d;
        }
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    lds[(threadIdx.x * V + e) * 2] = a[e];
    lds[(threadIdx.x * V + e) * 2 + 1] = b[e];
  }
  __syncthreads();
  if (!w.live || w.row0 != 0) return;
  double* out = p.part + ((w.n * p.slabs + w.slab) * (int64_t)p.channels + w.c) * 2;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    for (int r = 1; r < p.rows_at_once; ++r) {
      a[e] += lds[((threadIdx.x + r * p.lanes) * V + e) * 2];
      b[e] += lds[((threadIdx.x + r * p.lanes) * V + e) * 2 + 1];
    }
    out[2 * e] = a[e];
    out[2 * e + 1] = b[e];
  }
}

// The slabs' sums of one group, in a fixed order: mean and rstd, or (BWD) the two averages of the backward pass.
template <typename T, bool BWD>
__global__ __launch_bounds__(64) void group_fold(Args<T> p) {
  uint32_t g;
  const int64_t n = p.groups_div.divmod(blockIdx.x, g);
  double a = 0.0, b = 0.0;
  const double* part = p.part + (n * p.slabs * (int64_t)p.channels + (int64_t)g * p.per) * 2;
  const uint32_t total = (uint32_t)p.slabs * (uint32_t)p.per;
  for (uint32_t i = threadIdx.x; i < total; i += 64) {
    uint32_t c;
    const uint32_t slab = p.per_div.divmod(i, c);
    const double* at = part + ((int64_t)slab * p.channels + c) * 2;
    const double w = (BWD && p.weight) ? (double)p.weight[g * p.per + c] : 1.0;
    a += at[0] * w;
    b += at[1] * w;
  }
  for (int d = 32; d >= 1; d >>= 1) { a += __shfl_xor(a, d, 64); b += __shfl_xor(b, d, 64); }
  if (threadIdx.x) return;
  const double count = (double)p.spatial * (double)p.per;
  const int64_t at = n * p.groups + g;
  if constexpr (BWD) {
    p.coef[2 * at] = (T)(a / count);
    p.coef[2 * at + 1] = (T)(b / count);
  } else {
    const double m = a / count;
    double var = b / count - m * m;
    if (var < 0.0) var = 0.0;
    p.mean[at] = (T)((double)p.x[n * p.x_n + (int64_t)g * p.per] + m);
    p.rstd[at] = (T)(1.0 / sqrt(var + (double)p.eps));
  }
}

// dweight and dbias of 16 channels: 16 lanes side by side, 16 of them over the slabs, folded through LDS.
template <typename T>
__global__ __launch_bounds__(256) void channel_fold(Args<T> p, int64_t parts) {
  __shared__ double lds[256][2];
  const int c = (int)blockIdx.x * 16 + ((int)threadIdx.x & 15), k = (int)threadIdx.x >> 4;
  double a = 0.0, b = 0.0;
  if (c < p.channels) {
#pragma unroll 4
    for (int64_t i = k; i < parts; i += 16) {
      const double* at = p.part + (i * p.channels + c) * 2;
      a += at[0];
      b += at[1];
    }
  }
  lds[threadIdx.x][0] = a;
  lds[threadIdx.x][1] = b;
  __syncthreads();
  if (k != 0 || c >= p.channels) return;
  for (int r = 1; r < 16; ++r) { a += lds[threadIdx.x + 16 * r][0]; b += lds[threadIdx.x + 16 * r][1]; }
  if (p.dweight) p.dweight[c] = (T)(p.add ? (double)p.dweight[c] + b : b);
  if (p.dbias) p.dbias[c] = (T)(p.add ? (double)p.dbias[c] + a : a);
}

// Second pass over the slabs: y from mean and rstd, or (BWD) dx from the averages too.
template <typename T, int V, bool BWD, int ACT>
__global__ __launch_bounds__(256) void slab_apply(Args<T> p) {
  typedef typename Vec<T, V>::type vec_t;
  const Place w = place<T, V>(p);
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
    const vec_t xv = *(const vec_t*)(p.x + w.n * p.x_n + s * p.x_s + w.c);
    vec_t out;
    if constexpr (BWD) {
      const vec_t dv = *(const vec_t*)(p.dy + w.n * p.dy_n + s * p.dy_s + w.c);
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

// How a team covers a group of `units` vectors; 0 when it does not fit.
static int team_lanes(int64_t units) {
  for (int l = 8; l <= 64; l *= 2)
    if (units <= (int64_t)l * 4) return l;      // four vectors in flight for a lane
  if (units <= 256 * kUnits) return 256;
  return 0;
}

template <typename T> static void set_slabs(Args<T>& p, int V, int64_t rows, int64_t samples) {
  const int cv = p.channels / V;
  p.tiles = (cv + 255) / 256;
  p.lanes = cv < 256 ? cv : 256;
  p.rows_at_once = 256 / p.lanes;
  // a few workgroups for every CU, of at least eight rows for each lane
  int64_t slabs = ((int64_t)num_cus() * 8 + samples * p.tiles - 1) / (samples * p.tiles);
  const int64_t most = (rows + p.rows_at_once * 8 - 1) / (p.rows_at_once * 8);
  if (slabs > most) slabs = most;
  if (slabs < 1) slabs = 1;
  p.rows_per_slab = (rows + slabs - 1) / slabs;
  p.slabs = (int)((rows + p.rows_per_slab - 1) / p.rows_per_slab);
  p.tiles_div = FastDiv((uint32_t)p.tiles);
  p.slabs_div = FastDiv((uint32_t)p.slabs);
}

#define AM_GN_LAUNCH(KERNEL, V_, GRID, ...)                                                                         \
  do {                                                                                                              \
    const dim3 grid_((unsigned)(GRID)), block_(256);                                                                \
    if (V_ > 1) hipLaunchKernelGGL((KERNEL<T, W, __VA_ARGS__>), grid_, block_, 0, stream(), p);                      \
    else hipLaunchKernelGGL((KERNEL<T, 1, __VA_ARGS__>), grid_, block_, 0, stream(), p);                             \
  } while (0)

constexpr size_t kMostScratch = (size_t)256 << 20;

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

template <typename T, int ACT, bool BWD>
static int team_pass(Args<T> p, int V, int lanes, int units) {
  constexpr int W = 16 / (int)sizeof(T);
  const int64_t teams_per_wg = 256 / lanes;
  // at most 2^30 workgroups a launch
  const int64_t per_launch = (((int64_t)1 << 30) * teams_per_wg) / p.groups;
  const Args<T> all = p;
  for (int64_t n = 0; n < all.batch; n += per_launch) {
    p.nc = all.batch - n < per_launch ? all.batch - n : per_launch;
    p.x = all.x + n * p.x_n;
    p.y = all.y + n * p.y_n;
    if (BWD) p.dy = all.dy + n * p.dy_n;
    if (all.mean) { p.mean = all.mean + n * p.groups; p.rstd = all.rstd + n * p.groups; }
    const dim3 grid((unsigned)((p.nc * p.groups + teams_per_wg - 1) / teams_per_wg)), block(256);
    if (lanes == 256) {
      if constexpr (BWD) {
        if (V > 1) hipLaunchKernelGGL((team_backward<T, W, true, ACT>), grid, block, 0, stream(), p, lanes, units);
        else hipLaunchKernelGGL((team_backward<T, 1, true, ACT>), grid, block, 0, stream(), p, lanes, units);
      } else {
        if (V > 1) hipLaunchKernelGGL((team_forward<T, W, true, ACT>), grid, block, 0, stream(), p, lanes, units);
        else hipLaunchKernelGGL((team_forward<T, 1, true, ACT>), grid, block, 0, stream(), p, lanes, units);
      }
    } else {
      if constexpr (BWD) {
        if (V > 1) hipLaunchKernelGGL((team_backward<T, W, false, ACT>), grid, block, 0, stream(), p, lanes, units);
        else hipLaunchKernelGGL((team_backward<T, 1, false, ACT>), grid, block, 0, stream(), p, lanes, units);
      } else {
        if (V > 1) hipLaunchKernelGGL((team_forward<T, W, false, ACT>), grid, block, 0, stream(), p, lanes, units);
        else hipLaunchKernelGGL((team_forward<T, 1, false, ACT>), grid, block, 0, stream(), p, lanes, units);
      }
    }
    AM_TRY(check_launch("group norm of teams"));
  }
  return AM_OK;
}

template <typename T, int ACT>
static int forward(Args<T> p) {
  constexpr int W = 16 / (int)sizeof(T);
  const bool aligned = fits<T>(p.x, p.x_n, p.x_s, p.batch, p.spatial) && fits<T>(p.y, p.y_n, p.y_s, p.batch, p.spatial);
  {
    const int V = aligned && p.per % W == 0 ? W : 1;
    const int64_t upr = p.per / V;
    const int lanes = p.spatial <= 256 * kUnits ? team_lanes(p.spatial * upr) : 0;
    if (lanes) {
      p.units_div = FastDiv((uint32_t)upr);
      return team_pass<T, ACT, false>(p, V, lanes, (int)(p.spatial * upr));
    }
  }
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
  int64_t nc = (int64_t)(kMostScratch / per_sample);
  if (nc < 1) nc = 1;
  if (nc > p.batch) nc = p.batch;
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
    AM_GN_LAUNCH(slab_sums, V, wgs, false, false, ACT);
    AM_TRY(check_launch("slab_sums"));
    hipLaunchKernelGGL((group_fold<T, false>), dim3((unsigned)(p.nc * p.groups)), dim3(64), 0, stream(), p);
    AM_TRY(check_launch("group_fold"));
    AM_GN_LAUNCH(slab_apply, V, wgs, false, ACT);
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
  const int V = aligned && p.channels % W == 0 ? W : 1;
  const Args<T> all = p;
  Scratch part;
  const int TV = aligned && p.per % W == 0 ? W : 1;
  const int64_t upr = p.per / TV;
  const int lanes = p.spatial <= 256 * kUnits ? team_lanes(p.spatial * upr) : 0;
  if (lanes) {
    p.units_div = FastDiv((uint32_t)upr);
    AM_TRY((team_pass<T, ACT, true>(p, TV, lanes, (int)(p.spatial * upr))));
    if (!params) return AM_OK;
    p.nc = p.batch;
    set_slabs(p, V, p.batch * p.spatial, 1);
    AM_TRY(part.take((size_t)p.slabs * p.channels * 2 * sizeof(double)));
    p.part = (double*)part.p;
    AM_GN_LAUNCH(slab_sums, V, (int64_t)p.slabs * p.tiles, true, true, ACT);
    AM_TRY(check_launch("slab_sums"));
    hipLaunchKernelGGL((channel_fold<T>), dim3((unsigned)((p.channels + 15) / 16)), dim3(256), 0, stream(), p, (int64_t)p.slabs);
    return check_launch("channel_fold");
  }
  set_slabs(p, V, p.spatial, p.batch);
  const size_t per_sample = (size_t)p.slabs * p.channels * 2 * sizeof(double);
  int64_t nc = (int64_t)(kMostScratch / per_sample);
  if (nc < 1) nc = 1;
  if (nc > p.batch) nc = p.batch;
  const size_t coef_bytes = (size_t)nc * p.groups * 2 * sizeof(T);
  const size_t part_bytes = per_sample * (size_t)nc;
  AM_TRY(part.take(part_bytes + coef_bytes));
  p.part = (double*)part.p;
  p.coef = (T*)((char*)part.p + part_bytes);
  for (int64_t n = 0; n < all.batch; n += nc) {
    p.nc = all.batch - n < nc ? all.batch - n : nc;
    p.x = all.x + n * p.x_n;
    p.y = all.y + n * p.y_n;
    p.dy = all.dy + n * p.dy_n;
    p.mean = all.mean + n * p.groups;
    p.rstd = all.rstd + n * p.groups;
    const int64_t wgs = p.nc * p.slabs * p.tiles;
    AM_GN_LAUNCH(slab_sums, V, wgs, true, false, ACT);
    AM_TRY(check_launch("slab_sums"));
    hipLaunchKernelGGL((group_fold<T, true>), dim3((unsigned)(p.nc * p.groups)), dim3(64), 0, stream(), p);
    AM_TRY(check_launch("group_fold"));
    if (params) {
      p.add = n > 0;
      hipLaunchKernelGGL((channel_fold<T>), dim3((unsigned)((p.channels + 15) / 16)), dim3(256), 0, stream(), p, p.nc * p.slabs);
      AM_TRY(check_launch("channel_fold"));
    }
    AM_GN_LAUNCH(slab_apply, V, wgs, true, ACT);
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
