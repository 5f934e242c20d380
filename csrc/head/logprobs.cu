// Operators on the logits of a language-model head, x [rows, V], z = x / temperature, lse = log sum exp z,
// p = exp(z - lse):
//   * log-probabilities z_y - lse of given tokens y, the entropy H = -sum p (z - lse), the k most likely tokens;
//   * their gradient;
//   * the divergence from a teacher that is known by its top log-probabilities, with its gradient.
// All three are bound by the bytes of the logits. Statistics are held in 32 bits, relative to the row's maximum:
// with d_j = (x_j - max) log2(e) / t, l = sum 2^d, s = sum 2^d d:   z_j - lse = ln 2 (d_j - log2 l),
// H = ln 2 (log2 l - s / l), in which both terms are >= 0, so nothing cancels. (max, l) is what the gradient needs.
// The few scalars of a row are put together in 64 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include "../common/ptx.cuh"
#include "logprobs.h"

namespace zx {

namespace {

constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr double kLog2e = 1.442695040888963407359924681002;
constexpr int kThreads = 512;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }

__device__ __forceinline__ float inf_f() { return __int_as_float(0x7f800000); }
__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }
// Comparisons on the bits: the build's fast-math flag lets the compiler assume nothing about them, but says so.
__device__ __forceinline__ bool is_nan(float x) { return (__float_as_uint(x) & 0x7fffffffu) > 0x7f800000u; }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ int64_t load_id(const IdArray& a, size_t i) {
  return a.wide ? reinterpret_cast<const int64_t*>(a.p)[i] : (int64_t) reinterpret_cast<const int32_t*>(a.p)[i];
}

// Whole numbers in the order of the floats (-0 as +0), the column below: a larger key is the better alternative.
__device__ __forceinline__ uint64_t alt_key(float x, int col) {
  const uint32_t b = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t o = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  return ((uint64_t)o << 32) | (uint32_t)(0xffffffffu - (uint32_t)col);
}
__device__ __forceinline__ float key_value(uint64_t key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

template <class Op, class T>
__device__ T block_reduce(T v, T identity, Op op, T* s) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (lane == 0) s[warp] = v;
  __syncthreads();
  v = lane < (int)(blockDim.x >> 5) ? s[lane] : identity;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
struct MaxNan {   // a NaN wins
  __device__ float operator()(float a, float b) const { return is_nan(a) ? a : (is_nan(b) ? b : fmaxf(a, b)); }
};
struct Max64 {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};
struct Sum {
  __device__ float operator()(float a, float b) const { return a + b; }
};

// 2^d below this is nothing in 32 bits; keeps 0 * -inf out of s.
constexpr float kLeast = -1000.f;

template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_fwd_kernel(LogprobsArgs a) {
  __shared__ float sf[32];
  __shared__ uint64_t sk[32];
  const int row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  const int K = a.top_k;
  int64_t y = -1;
  if (a.targets.p != nullptr) {
    y = load_id(a.targets, row);
    if (y < 0 || y >= a.V) {   // left out
      if (threadIdx.x == 0) {
        a.logprobs[row] = 0.f;
        a.entropy[row] = 0.f;
        a.stats[row * 2] = a.stats[row * 2 + 1] = 0.f;
      }
      for (int k = threadIdx.x; k < K; k += blockDim.x) {
        a.top_logprobs[(size_t)row * K + k] = -inf_f();
        a.top_ids[(size_t)row * K + k] = -1;
      }
      return;
    }
  }
  float m = -inf_f();
  for (int j = threadIdx.x; j < a.V; j += blockDim.x) m = MaxNan()(m, to_f(x[j]));
  m = block_reduce(m, -inf_f(), MaxNan(), sf);
  const float c2 = (float)(kLog2e / (double)a.temperature);
  const bool bad = is_nan(m) || m == inf_f();   // no distribution
  const bool empty = m == -inf_f();             // nothing is left
  float l = 0.f, s = 0.f;
  if (!bad && !empty) {
    for (int j = threadIdx.x; j < a.V; j += blockDim.x) {
      const float d = fmaxf((to_f(x[j]) - m) * c2, kLeast);
      const float e = ex2(d);
      l += e;
      s += e * d;
    }
    l = block_reduce(l, 0.f, Sum(), sf);
    s = block_reduce(s, 0.f, Sum(), sf);
  }
  const double log_l = log((double)l);
  auto logprob = [&](float v) {
    if (bad) return nan_f();
    if (empty) return -inf_f();
    return (float)(((double)v - (double)m) / (double)a.temperature - log_l);
  };
  if (threadIdx.x == 0) {
    a.entropy[row] = bad ? nan_f() : (empty ? 0.f : (float)(log_l - kLn2 * (double)s / (double)l));
    a.stats[row * 2] = m;
    a.stats[row * 2 + 1] = bad ? nan_f() : l;
    if (y >= 0) a.logprobs[row] = logprob(to_f(x[y]));
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < K; ++k) {
    uint64_t best = 0;
    if (!bad && !empty) {
      for (int j = threadIdx.x; j < a.V; j += blockDim.x) {
        const float v = to_f(x[j]);
        const uint64_t key = alt_key(v, j);
        if (v > -inf_f() && key < last && key > best) best = key;
      }
      best = block_reduce(best, (uint64_t)0, Max64(), sk);
    }
    if (threadIdx.x == 0) {
      const bool none = best == 0;
      a.top_ids[(size_t)row * K + k] = none ? -1 : (int64_t)(0xffffffffu - (uint32_t)best);
      a.top_logprobs[(size_t)row * K + k] =
          bad ? nan_f() : (none ? -inf_f() : logprob(key_value(best)));
    }
    last = best;
  }
}

// Gradient of one row. The columns named by the target and the alternatives get their own coefficients: their
// logits are read before anything is written (the gradient may replace the logits) and written last.
template <class T>
__global__ void __launch_bounds__(kThreads) logprobs_bwd_kernel(LogprobsArgs a) {
  __shared__ int s_id[kHeadMaxTop + 1];
  __shared__ float s_c[kHeadMaxTop + 1];
  const int row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  T* dx = reinterpret_cast<T*>(a.d_logits) + (size_t)row * a.d_ld;
  const float m = a.stats[row * 2], l = a.stats[row * 2 + 1];
  const int64_t y = a.targets.p != nullptr ? load_id(a.targets, row) : -1;
  if (l == 0.f) {   // left out, or nothing is left
    for (int j = threadIdx.x; j < a.V; j += blockDim.x) from_f(0.f, dx[j]);
    return;
  }
  const int K = a.d_top != nullptr ? a.top_k : 0;
  for (int k = threadIdx.x; k <= K; k += blockDim.x) {
    int id = -1;
    float c = 0.f;
    if (k < K) {
      const int64_t i = a.top_ids[(size_t)row * K + k];
      if (i >= 0 && i < a.V) { id = (int)i; c = a.d_top[(size_t)row * K + k]; }
    } else if (y >= 0 && y < a.V && a.d_logprobs != nullptr) {
      id = (int)y;
      c = a.d_logprobs[row];
    }
    s_id[k] = id;
    s_c[k] = c;
  }
  __syncthreads();
  float g = 0.f;
  for (int k = 0; k <= K; ++k) g += s_c[k];
  const float h = a.d_entropy != nullptr ? a.d_entropy[row] : 0.f;
  const float H = a.entropy[row];
  const float it = 1.f / a.temperature, c2 = (float)(kLog2e / (double)a.temperature);
  const float inv_l = 1.f / l, H_l = H - (float)log((double)l);
  auto dense = [&](float v) {
    const float d = fmaxf((v - m) * c2, kLeast);
    const float p = is_nan(v) ? v : ex2(d) * inv_l;
    return -p * (g + h * (d * (float)kLn2 + H_l));
  };
  float own = 0.f;
  int own_id = -1;
  if ((int)threadIdx.x <= K && s_id[threadIdx.x] >= 0) {
    own_id = s_id[threadIdx.x];
    own = dense(to_f(x[own_id]));
    for (int k = 0; k <= K; ++k)
      if (s_id[k] == own_id) own += s_c[k];
  }
  __syncthreads();
  for (int j = threadIdx.x; j < a.V; j += blockDim.x) from_f(dense(to_f(x[j])) * it, dx[j]);
  __syncthreads();
  if (own_id >= 0) from_f(own * it, dx[own_id]);
}

__device__ __forceinline__ float load_value(const void* p, int type, size_t i) {
  if (type == LOGIT_BF16) return to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (type == LOGIT_FP16) return to_f(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}

// MODE 0: loss and stats; 1: gradient from stats; 2: loss and gradient.
// The columns of the teacher's tokens are kept apart (one bit a column in shared memory): the sum over all others is
// taken relative to their own maximum, so that the mass p_rest outside keeps its digits when the
// teacher's tokens have nearly all of it. stats = (maximum outside, coefficient of 2^d outside, maximum, 1 / l); the
// last is -1 for a row that is left out.
template <class T, int MODE>
__global__ void __launch_bounds__(kThreads) distill_kernel(DistillArgs a) {
  extern __shared__ uint32_t s_bits[];
  __shared__ float sf[32];
  __shared__ int s_id[kHeadMaxTop];
  __shared__ float s_v[kHeadMaxTop];
  const int row = blockIdx.x, K = a.K, tid = threadIdx.x;
  const T* x = reinterpret_cast<const T*>(a.logits) + (size_t)row * a.ld;
  T* dx = MODE ? reinterpret_cast<T*>(a.d_logits) + (size_t)row * a.d_ld : nullptr;
  const int words = (a.V + 31) / 32;
  for (int j = tid; j < words; j += blockDim.x) s_bits[j] = 0;
  if (tid < kHeadMaxTop) {
    int id = -1;
    float v = -inf_f();
    if (tid < K) {
      const int64_t i = load_id(a.ids, (size_t)row * K + tid);
      if (i >= 0 && i < a.V) { id = (int)i; v = load_value(a.values, a.value_type, (size_t)row * K + tid); }
    }
    s_id[tid] = id;
    s_v[tid] = v;
  }
  __syncthreads();
  float vm = -inf_f(), q_sum = 0.f;
  bool any = false;
  for (int k = 0; k < K; ++k) {
    vm = MaxNan()(vm, s_v[k]);
    any |= s_id[k] >= 0;
  }
  const float vbase = a.bucket ? 0.f : vm;
  any = any && (a.bucket || vm != -inf_f());
  if (!any) {
    if (MODE != 1 && tid == 0) {
      a.loss[row] = 0.f;
      if (MODE == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(0.f, 0.f, 0.f, -1.f);
    }
    if (MODE) for (int j = tid; j < a.V; j += blockDim.x) from_f(0.f, dx[j]);
    return;
  }
  for (int k = 0; k < K; ++k) q_sum += ex2((s_v[k] - vbase) * (float)kLog2e);
  const float q_norm = a.bucket ? 1.f : 1.f / q_sum;
  const float q_rest = a.bucket ? fmaxf(0.f, 1.f - q_sum) : 0.f;
  // own entry: its logit, and whether it is the first with its token
  const float c2 = (float)(kLog2e / (double)a.temperature);
  int id = tid < K ? s_id[tid] : -1;
  bool first = id >= 0;
  float q = 0.f, q_all = 0.f, xi = 0.f;
  if (id >= 0) {
    xi = to_f(x[id]);
    for (int k = 0; k < K; ++k) {
      if (s_id[k] != id) continue;
      if (k < tid) first = false;
      q_all += ex2((s_v[k] - vbase) * (float)kLog2e) * q_norm;
    }
    q = ex2((s_v[tid] - vbase) * (float)kLog2e) * q_norm;
    if (first) atomicOr(&s_bits[id >> 5], 1u << (id & 31));
  }
  __syncthreads();
  float mr, coef, m, inv_l;
  if (MODE == 1) {
    const float4 st = reinterpret_cast<const float4*>(a.stats)[row];
    mr = st.x; coef = st.y; m = st.z; inv_l = st.w;
  } else {
    mr = -inf_f();
    for (int j = tid; j < a.V; j += blockDim.x)
      if (!(s_bits[j >> 5] >> (j & 31) & 1)) mr = MaxNan()(mr, to_f(x[j]));
    mr = block_reduce(mr, -inf_f(), MaxNan(), sf);
    m = block_reduce(id >= 0 ? xi : -inf_f(), -inf_f(), MaxNan(), sf);
    m = MaxNan()(mr, m);
    const bool rest = mr != -inf_f();
    float lr = 0.f;
    if (rest)
      for (int j = tid; j < a.V; j += blockDim.x)
        if (!(s_bits[j >> 5] >> (j & 31) & 1)) lr += ex2((to_f(x[j]) - mr) * c2);
    lr = block_reduce(lr, 0.f, Sum(), sf);
    float lt = first && xi != -inf_f() ? ex2((xi - m) * c2) : 0.f;
    lt = block_reduce(lt, 0.f, Sum(), sf);
    const float share = rest ? ex2((mr - m) * c2) : 0.f;
    const float l = lt + lr * share;
    const double log_l = log((double)l);
    float part = 0.f;
    if (id >= 0 && q != 0.f) {
      const double lp = xi == -inf_f() ? -(double)inf_f() : ((double)xi - (double)m) / (double)a.temperature - log_l;
      part = (float)((double)q * (log((double)q) - lp));
    }
    float loss = block_reduce(part, 0.f, Sum(), sf);
    if (q_rest > 0.f && rest) {
      const double lp = ((double)mr - (double)m) / (double)a.temperature + log((double)lr) - log_l;
      loss += (float)((double)q_rest * (log((double)q_rest) - lp));
    }
    inv_l = l == 0.f ? 0.f : 1.f / l;
    coef = rest ? share * inv_l - q_rest / lr : 0.f;
    if (is_nan(m) || m == inf_f()) loss = coef = inv_l = nan_f();   // no distribution
    if (tid == 0) {
      a.loss[row] = loss;
      if (MODE == 0) reinterpret_cast<float4*>(a.stats)[row] = make_float4(mr, coef, m, inv_l);
    }
  }
  if (MODE == 0) return;
  const float w = (MODE == 1 ? a.d_loss[row] : a.grad_scale) / a.temperature;
  const float p = inv_l * (xi == -inf_f() ? 0.f : ex2((xi - m) * c2));
  __syncthreads();
  for (int j = tid; j < a.V; j += blockDim.x) {
    const float v = to_f(x[j]);
    from_f(w * (v == -inf_f() ? 0.f * coef : coef * ex2((v - mr) * c2)), dx[j]);
  }
  __syncthreads();
  if (first) from_f(w * (p - q_all), dx[id]);
}

template <class F>
void by_type(int type, F f) {
  if (type == LOGIT_BF16) f(__nv_bfloat16());
  else if (type == LOGIT_FP16) f(__half());
  else f(float());
}

template <int MODE>
void launch_distill(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) {
    using T = decltype(t);
    const int smem = (a.V + 31) / 32 * 4;
    cudaFuncSetAttribute(distill_kernel<T, MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024);
    distill_kernel<T, MODE><<<a.rows, kThreads, smem, a.stream>>>(a);
  });
}

}  // namespace

void launch_token_logprobs_fwd(const LogprobsArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { logprobs_fwd_kernel<decltype(t)><<<a.rows, kThreads, 0, a.stream>>>(a); });
}
void launch_token_logprobs_bwd(const LogprobsArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { logprobs_bwd_kernel<decltype(t)><<<a.rows, kThreads, 0, a.stream>>>(a); });
}
void launch_distill_fwd(const DistillArgs& a) { launch_distill<0>(a); }
void launch_distill_bwd(const DistillArgs& a) { launch_distill<1>(a); }
void launch_distill_fwd_bwd(const DistillArgs& a) { launch_distill<2>(a); }

}  // namespace zx
