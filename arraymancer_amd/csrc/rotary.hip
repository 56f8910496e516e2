// Rotary positions: am_hip_rotary_*.
//
// The first `rot_dim` elements of every head are rot_dim / 2 pairs (a, b) - element i with element i + rot_dim / 2
// (AM_ROTARY_HALF) or element 2 i with 2 i + 1 (AM_ROTARY_INTERLEAVED) - and pair i of a token at position p turns by the
// angle p * frequency[i]:
//     (a, b) -> scale * (a cos - b sin, b cos + a sin)
// The rest of the head is copied. The inverse (and, the turn being orthogonal, the gradient) is the same with -sin.
//
// The angle depends on the token and the pair alone, so a lane keeps one 16-byte vector of pairs of one token, makes its
// sines and cosines once and walks over the heads with them. Positions of long texts reach 10^5 and more, where a float
// angle is off by 10^-2: for results of either type the angle is the product in double and sine and cosine are made in double,
// whose reduction loses nothing however far the angle, and rounded to the result's type once, scale included. (Against a float sine
// of an angle that double had reduced: [4, 2048, 32, 128] 44.6 -> 45.1 us; with one head to a token [16, 4096, 1, 64] 8.8 -> 10.7.)
#include "common.h"
#include "fastdiv.h"

namespace am {
namespace rotary {

template <typename T> struct Args {
  const T* x; int64_t x_b, x_t, x_h;
  T* out; int64_t o_b, o_t, o_h;
  const int64_t* positions; int64_t p_b, p_t;    // null: the token's index
  const double* freq;
  int64_t first;                                 // first token (of batch * tokens) of this launch
  uint32_t items;                                // work items of this launch
  FastDiv units, blocks, tokens;                 // units per head; head blocks per token; tokens per batch entry
  uint32_t turning;                              // units that turn, the others are copied
  int heads, heads_per_lane, half;               // half = rot_dim / 2
  T scale, sign;
};

template <bool NT, typename V> __device__ __forceinline__ V fetch(const V* p) {
  if constexpr (NT) return __builtin_nontemporal_load(p);
  else return *p;
}

// One lane per unit (V consecutive elements of a head, with AM_ROTARY_HALF also their V partners) of `heads_per_lane`
// heads of one token. VEC: V = 16 bytes; else one element (pair). NT: x is read past the caches (a tensor larger than they
// keep; [4, 2048, 32, 128] float32 interleaved 55.5 -> 44.3 us, halves 57 -> 51, but [3, 1023, 12, 80] float64, 24 MB, 9.5 -> 11.2).
template <typename T, bool VEC, bool INTERLEAVED, bool NT>
__global__ __launch_bounds__(256) void rotate(Args<T> p) {
  constexpr int V = VEC ? 16 / (int)sizeof(T) : (INTERLEAVED ? 2 : 1);
  constexpr int P = INTERLEAVED ? V / 2 : V;     // pairs per unit
  typedef T vec_t __attribute__((ext_vector_type(V)));
  const uint32_t i = blockIdx.x * 256u + threadIdx.x;
  if (i >= p.items) return;
  uint32_t u, hb, t;
  const uint32_t rest = p.units.divmod(i, u);
  const int64_t bt = p.first + p.blocks.divmod(rest, hb);
  const int64_t b = bt / p.tokens.d;             // (one 64-bit division per lane, by a launch constant)
  t = (uint32_t)(bt - b * p.tokens.d);
  const int h0 = (int)hb * p.heads_per_lane;
  const int h1 = h0 + p.heads_per_lane < p.heads ? h0 + p.heads_per_lane : p.heads;
  const T* x = p.x + b * p.x_b + (int64_t)t * p.x_t;
  T* out = p.out + b * p.o_b + (int64_t)t * p.o_t;
  if (u >= p.turning) {                          // behind the turning part
    const int at = 2 * p.half + (int)(u - p.turning) * (VEC ? V : 1);
    for (int h = h0; h < h1; ++h) {
      if constexpr (VEC) *(vec_t*)(out + h * p.o_h + at) = *(const vec_t*)(x + h * p.x_h + at);
      else out[h * p.o_h + at] = x[h * p.x_h + at];
    }
    return;
  }
  const double pos = p.positions ? (double)p.positions[b * p.p_b + (int64_t)t * p.p_t] : (double)t;
  T sn[P], cs[P];
#pragma unroll
  for (int e = 0; e < P; ++e) {
    double s, c;
    sincos(pos * p.freq[u * P + e], &s, &c);
    sn[e] = (T)(s * (double)p.scale * (double)p.sign);
    cs[e] = (T)(c * (double)p.scale);
  }
  const int at = (int)u * V;
#pragma unroll 4
  for (int h = h0; h < h1; ++h) {
    const T* xh = x + h * p.x_h + at;
    T* oh = out + h * p.o_h + at;
    if constexpr (INTERLEAVED) {
      T v[V];
      if constexpr (VEC) {
        const vec_t w = fetch<NT>((const vec_t*)xh);
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = w[e];
      } else { v[0] = xh[0]; v[1] = xh[1]; }
      vec_t r;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        r[2 * e] = v[2 * e] * cs[e] - v[2 * e + 1] * sn[e];
        r[2 * e + 1] = v[2 * e + 1] * cs[e] + v[2 * e] * sn[e];
      }
      if constexpr (VEC) *(vec_t*)oh = r;
      else { oh[0] = r[0]; oh[1] = r[1]; }
    } else {
      const vec_t a = fetch<NT>((const vec_t*)xh), c = fetch<NT>((const vec_t*)(xh + p.half));
      vec_t ra, rc;
#pragma unroll
      for (int e = 0; e < P; ++e) {
        ra[e] = a[e] * cs[e] - c[e] * sn[e];
        rc[e] = c[e] * cs[e] + a[e] * sn[e];
      }
      *(vec_t*)oh = ra;
      *(vec_t*)(oh + p.half) = rc;
    }
  }
}

template <typename T>
static int launch(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t dim, int64_t rot_dim, int layout, int inverse,
                  T scale, const int64_t* positions, int64_t p_b, int64_t p_t, const double* freq, const T* x, int64_t x_b,
                  int64_t x_t, int64_t x_h, T* out, int64_t o_b, int64_t o_t, int64_t o_h) {
  if (layout != AM_ROTARY_HALF && layout != AM_ROTARY_INTERLEAVED) return fail(AM_E_ARG, "%s: unknown layout %d", fn, layout);
  if (batch < 0 || tokens < 0 || heads < 0 || dim < 0) return fail(AM_E_SHAPE, "%s: negative extent", fn);
  if (rot_dim < 0 || rot_dim > dim || rot_dim % 2) return fail(AM_E_SHAPE, "%s: %lld turning elements in a head of %lld (an even number up to the head is needed)", fn, (long long)rot_dim, (long long)dim);
  if (batch == 0 || tokens == 0 || heads == 0 || dim == 0) return AM_OK;
  if (!x || !out || (rot_dim && !freq)) return fail(AM_E_ARG, "%s: null tensor pointer", fn);
  if (dim >= ((int64_t)1 << 24) || heads >= ((int64_t)1 << 24) || tokens >= ((int64_t)1 << 31)) return fail(AM_E_SHAPE, "%s: extent too large", fn);
  if ((heads > 1 && o_h == 0) || (tokens > 1 && o_t == 0) || (batch > 1 && o_b == 0)) return fail(AM_E_SHAPE, "%s: the result is a broadcast view", fn);
  AM_TRY(ensure_init());
  constexpr int64_t W = 16 / (int64_t)sizeof(T);
  const bool inter = layout == AM_ROTARY_INTERLEAVED;
  const bool same = x == out && x_b == o_b && x_t == o_t && x_h == o_h;   // in place: the rest of the head is there already
  auto fits = [&](const void* base, int64_t sb, int64_t st, int64_t sh) {
    return (uintptr_t)base % 16 == 0 && (sb % W == 0 || batch == 1) && (st % W == 0 || tokens == 1) && (sh % W == 0 || heads == 1);
  };
  const bool vec = (inter ? rot_dim % W == 0 : rot_dim % (2 * W) == 0) && (same || (dim - rot_dim) % W == 0) && fits(x, x_b, x_t, x_h) && fits(out, o_b, o_t, o_h);
  Args<T> p = {};
  p.x = x; p.x_b = x_b; p.x_t = x_t; p.x_h = x_h;
  p.out = out; p.o_b = o_b; p.o_t = o_t; p.o_h = o_h;
  p.positions = positions; p.p_b = p_b; p.p_t = p_t;
  p.freq = freq; p.scale = scale; p.sign = inverse ? (T)-1 : (T)1;
  p.heads = (int)heads; p.half = (int)(rot_dim / 2);
  const int64_t pairs_per_unit = vec ? (inter ? W / 2 : W) : 1;
  const int64_t turning = rot_dim / 2 / pairs_per_unit;
  const int64_t units = turning + (same ? 0 : (dim - rot_dim) / (vec ? W : 1));
  if (units == 0) return AM_OK;
  p.turning = (uint32_t)turning;
  p.units = FastDiv((uint32_t)units);
  p.tokens = FastDiv((uint32_t)tokens);
  // A lane's sines serve up to 8 heads where that leaves a few waves for every SIMD; fewer heads per lane where there
  // are few tokens.
  int64_t per = 8;
  const int64_t rows = batch * tokens;
  while (per > 1 && rows * units * ((heads + per - 1) / per) < (int64_t)num_cus() * 1024) per >>= 1;
  p.heads_per_lane = (int)per;
  const int64_t blocks = (heads + per - 1) / per;
  p.blocks = FastDiv((uint32_t)blocks);
  const bool nt = (double)rows * heads * dim * sizeof(T) > nt_threshold_bytes();
  const int64_t rows_per_launch = ((int64_t)1 << 30) / (units * blocks) + 1;
  if (units * blocks >= ((int64_t)1 << 30)) return fail(AM_E_SHAPE, "%s: extent too large", fn);
  for (int64_t r = 0; r < rows; r += rows_per_launch) {
    const int64_t n = rows - r < rows_per_launch ? rows - r : rows_per_launch;
    p.first = r;
    p.items = (uint32_t)(n * units * blocks);
    const dim3 grid((unsigned)((p.items + 255u) / 256u)), block(256);
    if (vec && inter && nt) hipLaunchKernelGGL((rotate<T, true, true, true>), grid, block, 0, stream(), p);
    else if (vec && inter) hipLaunchKernelGGL((rotate<T, true, true, false>), grid, block, 0, stream(), p);
    else if (vec && nt) hipLaunchKernelGGL((rotate<T, true, false, true>), grid, block, 0, stream(), p);
    else if (vec) hipLaunchKernelGGL((rotate<T, true, false, false>), grid, block, 0, stream(), p);
    else if (inter) hipLaunchKernelGGL((rotate<T, false, true, false>), grid, block, 0, stream(), p);
    else hipLaunchKernelGGL((rotate<T, false, false, false>), grid, block, 0, stream(), p);
    AM_TRY(check_launch("rotate"));
  }
  return AM_OK;
}

}  // namespace rotary
}  // namespace am

using namespace am;

extern "C" int am_hip_rotary_f32(int64_t batch, int64_t tokens, int64_t heads, int64_t dim, int64_t rot_dim, int layout, int inverse,
                                 float scale, const int64_t* positions, int64_t pos_b, int64_t pos_t, const double* frequencies,
                                 const float* x, int64_t x_b, int64_t x_t, int64_t x_h, float* out, int64_t out_b, int64_t out_t,
                                 int64_t out_h) {
  return rotary::launch<float>("am_hip_rotary_f32", batch, tokens, heads, dim, rot_dim, layout, inverse, scale, positions, pos_b, pos_t,
                               frequencies, x, x_b, x_t, x_h, out, out_b, out_t, out_h);
}
extern "C" int am_hip_rotary_f64(int64_t batch, int64_t tokens, int64_t heads, int64_t dim, int64_t rot_dim, int layout, int inverse,
                                 double scale, const int64_t* positions, int64_t pos_b, int64_t pos_t, const double* frequencies,
                                 const double* x, int64_t x_b, int64_t x_t, int64_t x_h, double* out, int64_t out_b, int64_t out_t,
                                 int64_t out_h) {
  return rotary::launch<double>("am_hip_rotary_f64", batch, tokens, heads, dim, rot_dim, layout, inverse, scale, positions, pos_b, pos_t,
                                frequencies, x, x_b, x_t, x_h, out, out_b, out_t, out_h);
}
