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
  int out_group, out_member;         // > 1: only heads h with h % group == member run, and out has heads / group of them
  bool add;                          // out is added to
  const T* s0; int64_t s0_b, s0_h, s0_r, s0_c;     // first state [da, dc], null: zeros
  T* s1; int64_t s1_b, s1_h, s1_r, s1_c;           // last state, null: not wanted
  T scale_a, scale_b;
  int da, dc;
  const T* log_decay;
  const int64_t* lengths;
  int64_t batch, tokens, heads;      // heads: of the state and of log_decay
};

__device__ __forceinline__ float dev_exp(float v) { return expf(v); }
__device__ __forceinline__ double dev_exp(double v) { return exp(v); }
// e^{g n}; e^0 also where g is -infinity
template <typename T> __device__ __forceinline__ T power(T g, int64_t n) { return n == 0 ? (T)1 : dev_exp(g * (T)n); }

// Token by token: a wavefront owns 16 columns of one head's state, a lane one column and R rows of it (rows
// R * (lane / 16) ...), so a token's output is a sum over registers and two butterflies. Right for any size; its time is
// the chain of tokens.
template <typename T, int R, bool BACK>
__global__ __launch_bounds__(64) void walk(Role<T> p) {
  const int64_t b = blockIdx.z;
  const int h = (int)blockIdx.y * p.out_group + p.out_member;
  const int lane = (int)threadIdx.x, col = (int)blockIdx.x * 16 + (lane & 15), r0 = (lane >> 4) * R;
  const bool live = col < p.dc;
  const int c = live ? col : p.dc - 1;
  int64_t n = p.tokens;
  if (p.lengths) { const int64_t l = p.lengths[b]; n = l < 0 ? 0 : (l < n ? l : n); }
  const T lam = dev_exp(p.log_decay[h]);
  const T* qa = p.a.p + b * p.a.b + (h / p.a.group) * p.a.h;
  const T* kb = p.b.p + b * p.b.b + (h / p.b.group) * p.b.h;
  const T* vc = p.c.p + b * p.c.b + (h / p.c.group) * p.c.h + c;
  T* out = p.out + b * p.o_b + (int64_t)blockIdx.y * p.o_h + c;
  T s[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + i;
    s[i] = (p.s0 && r < p.da) ? p.s0[b * p.s0_b + h * p.s0_h + r * p.s0_r + c * p.s0_c] : (T)0;
  }
  for (int64_t i = 0; i < n; ++i) {
    const int64_t t = BACK ? n - 1 - i : i;
    const T v = vc[t * p.c.t];
    T o = (T)0;
#pragma unroll
    for (int e = 0; e < R; ++e) {
      const int r = r0 + e;
      if (r < p.da) {
        const T kv = kb[t * p.b.t + r] * p.scale_b * v;
        if constexpr (BACK) s[e] += kv;
        else s[e] = s[e] * lam + kv;
        o += qa[t * p.a.t + r] * p.scale_a * s[e];
        if constexpr (BACK) s[e] *= lam;
      }
    }
    o += __shfl_xor(o, 16, 64);
    o += __shfl_xor(o, 32, 64);
    if (live && lane < 16) out[t * p.o_t] = p.add ? out[t * p.o_t] + o : o;
  }
  if (live && lane < 16 && !p.add)
    for (int64_t t = n; t < p.tokens; ++t) out[t * p.o_t] = (T)0;     // behind the sequence
  if (p.s1 && live) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int r = r0 + i;
      if (r < p.da) p.s1[b * p.s1_b + h * p.s1_h + r * p.s1_r + c * p.s1_c] = s[i];
    }
  }
}

template <typename T, bool BACK>
static int run_role(const Role<T>& p) {
  const int64_t heads = p.heads / p.out_group;
  const dim3 grid((unsigned)((p.dc + 15) / 16), (unsigned)heads, (unsigned)p.batch), block(64);
  if (p.da <= 64) hipLaunchKernelGGL((walk<T, 16, BACK>), grid, block, 0, stream(), p);
  else if (p.da <= 128) hipLaunchKernelGGL((walk<T, 32, BACK>), grid, block, 0, stream(), p);
  else hipLaunchKernelGGL((walk<T, 64, BACK>), grid, block, 0, stream(), p);
  return check_launch("walk");
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

constexpr int64_t kMostDim = 256;

static int check_sizes(const char* fn, int64_t batch, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t dk, int64_t dv) {
  if (batch < 0 || tokens < 0 || heads < 0 || kv_heads < 0) return fail(AM_E_SHAPE, "%s: negative extent", fn);
  if (dk < 1 || dv < 1 || dk > kMostDim || dv > kMostDim)
    return fail(AM_E_SHAPE, "%s: heads of %lld and %lld elements (1 .. %lld are supported)", fn, (long long)dk, (long long)dv, (long long)kMostDim);
  if (heads && (kv_heads < 1 || heads % kv_heads)) return fail(AM_E_SHAPE, "%s: %lld heads cannot share %lld key / value heads evenly", fn, (long long)heads, (long long)kv_heads);
  if (heads > 65535 || batch > 65535) return fail(AM_E_SHAPE, "%s: more than 65535 heads or batch entries", fn);
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
  p.out_group = 1;
  p.s0 = s0; p.s0_b = s0_b; p.s0_h = s0_h; p.s0_r = dv; p.s0_c = 1;
  p.s1 = s1; p.s1_b = s1_b; p.s1_h = s1_h; p.s1_r = dv; p.s1_c = 1;
  p.scale_a = scale; p.scale_b = (T)1;
  p.da = (int)dk; p.dc = (int)dv;
  p.log_decay = log_decay; p.lengths = lengths;
  p.batch = batch; p.tokens = tokens; p.heads = heads;
  return run_role<T, false>(p);
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
  p.out_group = 1;
  p.s0 = s0; p.s0_b = s0_b; p.s0_h = s0_h; p.s0_r = 1; p.s0_c = dv;
  p.scale_a = scale; p.scale_b = (T)1;
  p.da = (int)dv; p.dc = (int)dk;
  AM_TRY((run_role<T, false>(p)));
  // dv and dk: backwards; key / value heads that several heads share add up their shares one head after the other, in
  // the heads' order
  p.out_group = group;
  p.scale_a = (T)1; p.scale_b = scale;
  for (int m = 0; m < group; ++m) {
    p.out_member = m;
    p.add = m > 0;
    p.a = K; p.b = Q; p.c = G;
    p.out = dval.p; p.o_b = dval.b; p.o_t = dval.t; p.o_h = dval.h;
    p.s0 = gs; p.s0_b = gs_b; p.s0_h = gs_h; p.s0_r = dv; p.s0_c = 1;
    p.s1 = gs0; p.s1_b = gs0_b; p.s1_h = gs0_h; p.s1_r = dv; p.s1_c = 1;
    p.da = (int)dk; p.dc = (int)dv;
    AM_TRY((run_role<T, true>(p)));
    p.a = W; p.b = G; p.c = Q;
    p.out = dkey.p; p.o_b = dkey.b; p.o_t = dkey.t; p.o_h = dkey.h;
    p.s0_r = 1; p.s0_c = dv;
    p.s1 = nullptr;
    p.da = (int)dv; p.dc = (int)dk;
    AM_TRY((run_role<T, true>(p)));
  }
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
