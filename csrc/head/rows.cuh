// Rows of logits as the kernels of this directory see them: element types, 16-byte vectors, sums of exponentials.
//
// A row is walked in vectors of 16 bytes from the aligned address at or below its first logit ("virtual" vectors:
// those at the two ends may be partial, what they lack reads as -inf), so rows may start anywhere.
//
// Sums of exponentials are held in 32 bits relative to a maximum m of the row's logits: with c2 = log2(e) / temperature,
// 2^rel(x) with rel(x) = x c2 - ref(m), ref(m) = m c2 rounded. One fused multiply-add a logit; the rounding of ref(m) is
// in every term alike and cancels, as long as every reader of (m, sum) takes the same ref(m). It must be small beside 1,
// though: rel(m) is that rounding, and 2^rel(m) has to stay near 1. Where |m c2| is 2^20 or more (a row whose mask leaves
// large negative numbers only), rel(x) = (x - m) c2: two instructions, and ref(m) is the exact product.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include <algorithm>
#include "../common/ptx.cuh"
#include "logprobs.h"

namespace zx {

constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr double kLog2e = 1.442695040888963407359924681002;
// 2^d below this is nothing in 32 bits; keeps 0 * -inf out of the entropy.
constexpr float kLeast = -1000.f;

// ------------------------------------------------------------------------------------------
// Elements
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ void from_f(float v, float& o) { o = v; }
__device__ __forceinline__ void from_f(float v, __nv_bfloat16& o) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_f(float v, __half& o) { o = __float2half_rn(v); }

__device__ __forceinline__ float inf_f() { return __int_as_float(0x7f800000); }
__device__ __forceinline__ float nan_f() { return __int_as_float(0x7fffffff); }
__device__ __forceinline__ bool is_nan(float x) { return (__float_as_uint(x) & 0x7fffffffu) > 0x7f800000u; }
// No distribution: the row holds a NaN or +inf.
__device__ __forceinline__ bool is_bad(float m) { return is_nan(m) || m == inf_f(); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Maximum in which a NaN wins.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Two 32-bit floats in one register pair: one instruction does both.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

template <class T>
struct Elem;
template <>
struct Elem<__nv_bfloat16> {
  static constexpr int kPerWord = 2;
  static constexpr uint32_t kNegInf = 0xff80ff80u;
  static __device__ __forceinline__ uint32_t max_w(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint64_t wide(uint32_t w) {
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t narrow(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Elem<__half> {
  static constexpr int kPerWord = 2;
  static constexpr uint32_t kNegInf = 0xfc00fc00u;
  static __device__ __forceinline__ uint32_t max_w(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ uint64_t wide(uint32_t w) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return pair(f.x, f.y);
  }
  static __device__ __forceinline__ uint32_t narrow(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct Elem<float> {
  static constexpr int kPerWord = 1;
  static constexpr uint32_t kNegInf = 0xff800000u;
  static __device__ __forceinline__ uint32_t max_w(uint32_t a, uint32_t b) {
    return __float_as_uint(max_nan(__uint_as_float(a), __uint_as_float(b)));
  }
};

// The pairs of a 16-byte vector, in column order.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  static constexpr int kPairs = N / 2;
  static __device__ __forceinline__ uint64_t get(const uint4& v, int i) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    if constexpr (Elem<T>::kPerWord == 2) return Elem<T>::wide(w[i]);
    else return pair(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
  // Two results into the place of pair i.
  static __device__ __forceinline__ void put(uint4& v, int i, uint64_t ab) {
    float a, b;
    unpair(ab, a, b);
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
    if constexpr (Elem<T>::kPerWord == 2) {
      w[i] = Elem<T>::narrow(a, b);
    } else {
      w[2 * i] = __float_as_uint(a);
      w[2 * i + 1] = __float_as_uint(b);
    }
  }
  // Element i of a vector in registers.
  static __device__ __forceinline__ float one(const uint4& v, int i) {
    const int word = Elem<T>::kPerWord == 2 ? i >> 1 : i;
    const uint32_t a = word & 1 ? v.y : v.x, b = word & 1 ? v.w : v.z, w = word & 2 ? b : a;
    if constexpr (Elem<T>::kPerWord == 2) {
      float lo, hi;
      unpair(Elem<T>::wide(w), lo, hi);
      return i & 1 ? hi : lo;
    } else {
      return __uint_as_float(w);
    }
  }
  static __device__ __forceinline__ uint32_t max_w(const uint4& v) {
    return Elem<T>::max_w(Elem<T>::max_w(v.x, v.y), Elem<T>::max_w(v.z, v.w));
  }
  static __device__ __forceinline__ float max_of(uint32_t w) {
    if constexpr (Elem<T>::kPerWord == 2) {
      float a, b;
      unpair(Elem<T>::wide(w), a, b);
      return max_nan(a, b);
    } else {
      return __uint_as_float(w);
    }
  }
  static __device__ __forceinline__ uint4 nothing() {
    return make_uint4(Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf, Elem<T>::kNegInf);
  }
};

// ------------------------------------------------------------------------------------------
// Rows
// ------------------------------------------------------------------------------------------
template <class T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* x;
  int V, lead, first_full, end_full, vecs;   // whole vectors: [first_full, end_full), none if that is empty
  __device__ __forceinline__ Row(const void* p, size_t row, int64_t ld, int V_) : x(reinterpret_cast<const T*>(p) + row * ld), V(V_) {
    lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    first_full = lead > 0 ? 1 : 0;
    end_full = (lead + V) / N;
    vecs = (lead + V + N - 1) / N;
  }
  __device__ __forceinline__ int col(int i) const { return i * N - lead; }
  __device__ __forceinline__ int vec_of(int column) const { return (column + lead) / N; }
  __device__ __forceinline__ bool whole(int i) const { return i >= first_full && i < end_full; }
  __device__ __forceinline__ const uint4* at(int i) const { return reinterpret_cast<const uint4*>(x - lead) + i; }
  __device__ __forceinline__ uint4 edge(int i) const {
    uint4 v = Vec<T>::nothing();
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if ((unsigned)(col(i) + k) < (unsigned)V) e[k] = x[col(i) + k];
    return v;
  }
  // Vector i of those before end. Plain loads: the row may be overwritten by the same kernel later on.
  __device__ __forceinline__ uint4 load(int i, int end) const {
    if (whole(i) && i < end) return *at(i);
    return i < end ? edge(i) : Vec<T>::nothing();
  }
  // U vectors i, i + step, ... of a block whose first is i0; the check that all of them are whole is the block's.
  template <int U>
  __device__ __forceinline__ void load_group(uint4 (&v)[U], int i0, int i, int step, int end) const {
    if (i0 >= first_full && i0 + U * step <= min(end, end_full)) {
      const uint4* p = at(i);
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = p[u * step];
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) v[u] = load(i + u * step, end);
    }
  }
};

// A row of gradients; it may start at another address than the logits'.
template <class T>
struct OutRow {
  T* p;
  bool vectors;   // its 16-byte boundaries are the logits'
  __device__ __forceinline__ OutRow(void* base, size_t row, int64_t ld, const Row<T>& in) : p(reinterpret_cast<T*>(base) + row * ld) {
    vectors = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(in.x)) & 15) == 0;
  }
  __device__ __forceinline__ uint4* at(const Row<T>& in, int i) const { return reinterpret_cast<uint4*>(p - in.lead) + i; }
  __device__ __forceinline__ void store(const Row<T>& in, int i, const uint4& v) const {
    if (vectors && in.whole(i)) {
      *at(in, i) = v;
      return;
    }
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k)
      if ((unsigned)(in.col(i) + k) < (unsigned)in.V) p[in.col(i) + k] = e[k];
  }
};

__device__ __forceinline__ int64_t load_id(const IdArray& a, size_t i) {
  return a.wide ? reinterpret_cast<const int64_t*>(a.p)[i] : (int64_t) reinterpret_cast<const int32_t*>(a.p)[i];
}

// ------------------------------------------------------------------------------------------
// Exponentials relative to a maximum
// ------------------------------------------------------------------------------------------
__device__ __forceinline__ float scale2(float temperature) { return (float)(kLog2e / (double)temperature); }
__device__ __forceinline__ float ref2(float m, float c2) { return __fmul_rn(m, c2); }
constexpr float kFar = 1048576.f;
__device__ __forceinline__ bool is_far(float m, float c2) { return !(fabsf(ref2(m, c2)) < kFar); }
__device__ __forceinline__ double ref2_exact(float m, float c2) { return is_far(m, c2) ? (double)m * (double)c2 : (double)ref2(m, c2); }
__device__ __forceinline__ float rel2(float x, float m, float c2) {
  return is_far(m, c2) ? (x - m) * c2 : __fmaf_rn(x, c2, -ref2(m, c2));
}
__device__ __forceinline__ double rel2_exact(float x, float m, float c2) {
  return is_far(m, c2) ? ((double)x - (double)m) * (double)c2 : (double)x * (double)c2 - (double)ref2(m, c2);
}
// What sums relative to m are worth relative to M >= m: 2^gap.
__device__ __forceinline__ double gap2_exact(float m, float M, float c2) {
  return m == M ? 0. : ref2_exact(m, c2) - ref2_exact(M, c2);
}
// Far from zero the rounded products may hide the gap, or be one where there is hardly any. Where M is nearer than
// plain_gap's limit, an m that is far has a gap beyond kLeast either way.
__device__ __forceinline__ bool plain_gap(float ref_M) { return fabsf(ref_M) < kFar - 2048.f; }
__device__ __forceinline__ float gap2_plain(float m, float ref_M, float c2) {
  return fmaxf(ref2(m, c2) - ref_M, kLeast);   // (the maximum of a NaN and kLeast is kLeast)
}
__device__ __forceinline__ float gap2_far(float m, float M, float c2) {
  auto rounding = [&](float x) { return is_far(x, c2) ? 0.f : __fmaf_rn(x, c2, -ref2(x, c2)); };
  return m == M ? 0.f : fmaxf(__fmaf_rn(m - M, c2, rounding(M) - rounding(m)), kLeast);
}
__device__ __forceinline__ float gap2(float m, float M, float c2) {
  const float R = ref2(M, c2);
  return plain_gap(R) ? gap2_plain(m, R, c2) : gap2_far(m, M, c2);
}

// rel2 of two logits at once; `Far` as is_far(m, c2).
template <bool Far>
struct Rel2 {
  uint64_t c22, a;
  __device__ __forceinline__ Rel2(float m, float c2) : c22(pair(c2, c2)) {
    const float s = Far ? -m : -ref2(m, c2);
    a = pair(s, s);
  }
  __device__ __forceinline__ uint64_t operator()(uint64_t x) const { return Far ? mul2(add2(x, a), c22) : fma2(x, c22, a); }
};

// ------------------------------------------------------------------------------------------
// Warps and clusters
// ------------------------------------------------------------------------------------------
// Over groups of W neighbouring lanes.
template <int W = 32>
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int W = 32>
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

constexpr int kMaxCluster = 8;   // what every device takes

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_to_cta(void* p, uint32_t rank, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(map_to_cta(p, rank)), "f"(v) : "memory");
}
__device__ __forceinline__ void store_to_cta(void* p, uint32_t rank, uint64_t v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(map_to_cta(p, rank)), "l"(v) : "memory");
}

// bytes: whole 16-byte vectors of one row.
__device__ __forceinline__ void prefetch_l2(const uint4* p, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"(bytes) : "memory");
}

// ------------------------------------------------------------------------------------------
// Launches
// ------------------------------------------------------------------------------------------
template <class F>
void by_type(int type, F f) {
  if (type == LOGIT_BF16) f(__nv_bfloat16());
  else if (type == LOGIT_FP16) f(__half());
  else f(float());
}
// Most virtual vectors that a row can have.
template <class T>
int most_vecs(const void* p, int64_t ld, int rows, int V) {
  const bool aligned = (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (rows == 1 || ld * (int64_t)sizeof(T) % 16 == 0);
  constexpr int N = 16 / sizeof(T);
  return aligned ? (V + N - 1) / N : (V + 2 * (N - 1)) / N;
}
template <class... P, class... A>
void launch(void (*kernel)(P...), int rows, int blocks_a_row, bool cluster, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  // (a grid holds 2^31 - 1 blocks: a launch of more is refused)
  cfg.gridDim = dim3((unsigned)std::min<int64_t>((int64_t)rows * blocks_a_row, UINT32_MAX));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks_a_row;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster && blocks_a_row > 1 ? 1 : 0;
  // 48 KB go without asking, the kernel's own arrays included. The limit is raised, never lowered: launches of other sizes
  // rely on it.
  if (smem > 32 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace zx
