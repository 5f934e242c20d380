// Operators on the logits of a language-model head, x [rows, V], z = x / temperature, lse = log sum exp z,
// p = exp(z - lse):
//   * log-probabilities z_y - lse of given tokens y, the entropy H = -sum p (z - lse), the k most likely tokens;
//   * their gradient;
//   * the divergence from a teacher that is known by its top log-probabilities, with its gradient.
// All three are bound by the bytes of the logits. Statistics are held in 32 bits, relative to a maximum:
// with d_j = (x_j - max) log2(e) / t, l = sum 2^d, s = sum 2^d d:   z_j - lse = ln 2 (d_j - log2 l),
// H = ln 2 (log2 l - s / l), in which both terms are >= 0, so nothing cancels. (max, l) is what the gradient needs.
// The few scalars of a row are put together in 64 bits.
//
// A row is walked in vectors of 16 bytes from the aligned address at or below its first logit ("virtual" vectors:
// those at the two ends may be partial, what they lack reads as -inf), so rows may start anywhere.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <float.h>
#include "../common/ptx.cuh"
#include "logprobs.h"

namespace zx {

namespace {

constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr double kLog2e = 1.442695040888963407359924681002;
// 2^d below this is nothing in 32 bits; keeps 0 * -inf out of the entropy.
constexpr float kLeast = -1000.f;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;

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
  static constexpr uint32_t kStep = 1u << 16;    // between two neighbours, as bits of fp32
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
  static constexpr uint32_t kStep = 1u << 13;
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
  static constexpr uint32_t kStep = 1;
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
  // element e becomes -inf where bit e of mask is set
  static __device__ __forceinline__ void drop(uint4& v, uint32_t mask) {
    uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (Elem<T>::kPerWord == 2) {
        const uint32_t m = ((mask >> (2 * i) & 1) ? 0xffffu : 0u) | ((mask >> (2 * i + 1) & 1) ? 0xffff0000u : 0u);
        w[i] = (w[i] & ~m) | (Elem<T>::kNegInf & m);
      } else {
        if (mask >> i & 1) w[i] = Elem<T>::kNegInf;
      }
    }
  }
};

// One row as virtual vectors.
template <class T>
struct Row {
  static constexpr int N = Vec<T>::N;
  const T* x;
  int V, lead, first_full, full, vecs;
  __device__ __forceinline__ Row(const void* p, size_t row, int64_t ld, int V_) : x(reinterpret_cast<const T*>(p) + row * ld), V(V_) {
    lead = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    first_full = lead > 0 ? 1 : 0;
    full = (lead + V) / N - first_full;          // whole vectors from first_full on (may be -1: inside one vector)
    vecs = (lead + V + N - 1) / N;
  }
  __device__ __forceinline__ int col(int i) const { return i * N - lead; }
  __device__ __forceinline__ bool whole(int i) const { return i >= first_full && i < first_full + full; }
  __device__ __forceinline__ const uint4* at(int i) const {
    return reinterpret_cast<const uint4*>(x - lead) + i;
  }
  __device__ __forceinline__ uint4 edge(int i) const {
    uint4 v = Vec<T>::nothing();
    T* e = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if ((unsigned)(col(i) + k) < (unsigned)V) e[k] = x[col(i) + k];
    return v;
  }
  // Plain loads: the row may be overwritten by the same kernel later on.
  __device__ __forceinline__ uint4 load(int i, int end) const {
    if (whole(i) && i < end) return *at(i);
    return i < end ? edge(i) : Vec<T>::nothing();
  }
};

__device__ __forceinline__ int64_t load_id(const IdArray& a, size_t i) {
  return a.wide ? reinterpret_cast<const int64_t*>(a.p)[i] : (int64_t) reinterpret_cast<const int32_t*>(a.p)[i];
}
__device__ __forceinline__ float load_value(const void* p, int type, size_t i) {
  if (type == LOGIT_BF16) return to_f(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (type == LOGIT_FP16) return to_f(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}

// Whole numbers in the order of the floats (-0 as +0); -inf is the smallest that occurs.
__device__ __forceinline__ uint32_t order_key(float x) {
  uint32_t b = __float_as_uint(x);
  b = b == 0x80000000u ? 0u : b;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
constexpr uint32_t kNegInfKey = 0x007fffffu;
__device__ __forceinline__ float key_value(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o); }
// The column below: a larger key is the better alternative, no two are alike, 0 is none.
__device__ __forceinline__ uint64_t alt_key(uint32_t o, int col) { return ((uint64_t)o << 32) | (0xffffffffu - (uint32_t)col); }
__device__ __forceinline__ int alt_col(uint64_t key) { return (int)(0xffffffffu - (uint32_t)key); }

// ------------------------------------------------------------------------------------------
// Clusters
// ------------------------------------------------------------------------------------------
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

// ------------------------------------------------------------------------------------------
// (maximum, sum of 2^d, sum of 2^d d): joining
// ------------------------------------------------------------------------------------------
struct Sums {
  float m, l, s;
};
// What a sum relative to m is worth relative to M >= m.
__device__ __forceinline__ void move_to(Sums& a, float M, float c2) {
  const float d = fmaxf((a.m - M) * c2, kLeast), f = ex2(d);
  a.s = f * (a.s + a.l * d);
  a.l *= f;
  a.m = M;
}
__device__ __forceinline__ Sums warp_join(Sums a, float c2) {
  float M = a.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = max_nan(M, __shfl_xor_sync(0xffffffffu, M, o));
  move_to(a, M, c2);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.l += __shfl_xor_sync(0xffffffffu, a.l, o);
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
  }
  return a;
}

// ------------------------------------------------------------------------------------------
// The k best of a set, in a block
// ------------------------------------------------------------------------------------------
constexpr int kCandidates = 1024;

struct TopShared {
  uint64_t list[kCandidates];
  uint64_t best[kHeadMaxTop];
  int count[80];           // one counter for each step of a search, so that a step takes one barrier
  uint32_t hist[256];
  int n, taken;
  uint32_t lo, hi;
  int warp[kWarps];
};

// Adds up every thread's share through counter i; a barrier.
__device__ __forceinline__ int block_count(TopShared& sh, int i, int mine) {
  mine = __reduce_add_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0 && mine) atomicAdd(&sh.count[i], mine);
  __syncthreads();
  return sh.count[i];
}

// A bound lo >= the given one with at least k members of the set at or above it, and few more. `share(bound)` counts a
// thread's members; hi lies above all. Needs count(lo) >= k at the start.
template <class Key, class Share>
__device__ __forceinline__ Key find_bound(TopShared& sh, Key lo, Key hi, Key step, int k, Share share) {
  const int slack = k / 4 + 4;
#pragma unroll 1
  for (int i = 0; i < 72 && hi - lo > step; ++i) {
    const Key mid = lo + (hi - lo) / 2;
    const int n = block_count(sh, i, share(mid));
    if (n < k) {
      hi = mid;
    } else {
      lo = mid;
      if (n <= k + slack) break;
    }
  }
  return lo;
}
__device__ __forceinline__ void clear_counts(TopShared& sh) {
  __syncthreads();
  for (int i = threadIdx.x; i < 80; i += blockDim.x) sh.count[i] = 0;
  __syncthreads();
}

// best[0 .. k) = the k largest of list[0 .. n), in order (0 where there are fewer): each finds its own place.
__device__ __forceinline__ void rank_list(TopShared& sh, int n, int k) {
  for (int i = threadIdx.x; i < k; i += blockDim.x) sh.best[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const uint64_t mine = sh.list[i];
    int r = 0;
    for (int j = 0; j < n; ++j) r += sh.list[j] > mine;
    if (r < k) sh.best[r] = mine;
  }
  __syncthreads();
}

// Any input, ties without end: the k-th largest value by its digits (four passes of 8 bits), then everything above it and
// the first of its equals in column order. Reads the vectors [v0, v1) of the row five times.
template <class T>
__device__ __noinline__ void select_exactly(TopShared& sh, const Row<T>& row, int v0, int v1, int k) {
  constexpr int N = Vec<T>::N;
  const int tid = threadIdx.x, lane = tid & 31;
  uint32_t prefix = 0, mask = 0;
  int need = k;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += blockDim.x) sh.hist[i] = 0;
    __syncthreads();
    for (int i = v0 + tid; i < v1 + 31; i += blockDim.x) {   // whole warps
      if (i - lane >= v1) break;
      const uint4 v = row.load(i, v1);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll 1
      for (int j = 0; j < N; ++j) {
        const uint32_t key = order_key(to_f(e[j]));
        const bool in = key > kNegInfKey && (key & mask) == prefix;
        const uint32_t digit = in ? (key >> shift & 255u) : 256u;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        if (in && (int)__ffs(same) - 1 == lane) atomicAdd(&sh.hist[digit], __popc(same));
      }
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, above = 0;
      for (; d > 0; --d) {
        if (above + (int)sh.hist[d] >= need) break;
        above += sh.hist[d];
      }
      sh.lo = d;
      sh.taken = above;
    }
    __syncthreads();
    prefix |= sh.lo << shift;
    mask |= 255u << shift;
    need -= sh.taken;
    __syncthreads();
  }
  if (prefix <= kNegInfKey) prefix = kNegInfKey;   // fewer than k: all that there are are above it
  if (tid == 0) sh.n = 0;
  int ties = 0;   // of those before this round's vectors
  __syncthreads();
  for (int base = v0; base < v1; base += blockDim.x) {
    const int i = base + tid;
    const uint4 v = row.load(i, v1);
    const T* e = reinterpret_cast<const T*>(&v);
    int equal = 0;
#pragma unroll 1
    for (int j = 0; j < N; ++j) {
      const uint32_t key = order_key(to_f(e[j]));
      if (key > prefix) sh.list[atomicAdd(&sh.n, 1)] = alt_key(key, row.col(i) + j);
      equal += key == prefix && key > kNegInfKey;
    }
    int before = equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    if (lane == 31) sh.warp[tid >> 5] = before;
    __syncthreads();
    int place = ties + before - equal, all = ties;
    for (int w = 0; w < (int)(blockDim.x >> 5); ++w) {
      if (w < (tid >> 5)) place += sh.warp[w];
      all += sh.warp[w];
    }
    for (int j = 0; j < N && place < need && equal > 0; ++j) {
      const uint32_t key = order_key(to_f(e[j]));
      if (key == prefix) {
        sh.list[atomicAdd(&sh.n, 1)] = alt_key(key, row.col(i) + j);
        ++place;
        --equal;
      }
    }
    ties = all;
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------
// Log-probabilities, entropy, alternatives: one pass over the row, by a block or by a cluster of them
// ------------------------------------------------------------------------------------------
constexpr int kUnroll = 4;    // vectors of a thread in flight

struct FwdShared {
  Sums part[kWarps];
  float cta[kMaxCluster][3];
  float m, log_l_hi, log_l_lo;
  int bad;
  uint32_t wmin[kWarps], wmax[kWarps];
};

// TOP: a thread keeps the maximum of each of its groups (kUnroll vectors) in shared memory. The k-th largest group
// maximum bounds the k-th largest logit from below, so only groups at or above it (about k of them) are read again.
template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprobs_fwd_kernel(LogprobsArgs a, int cluster, int steps) {
  constexpr int P = Vec<T>::kPairs;
  // TOP: TopShared, the keys of the cluster's blocks [cluster][k] (in the first block), the group maxima
  extern __shared__ __align__(16) unsigned char dynamic[];
  __shared__ FwdShared sh;
  TopShared& top = *reinterpret_cast<TopShared*>(dynamic);
  uint64_t* lists = reinterpret_cast<uint64_t*>(dynamic + sizeof(TopShared));
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  const int r = blockIdx.x / cluster, rank = blockIdx.x % cluster;
  const int K = a.top_k;
  if (cluster > 1) cluster_arrive();
  const Row<T> row(a.logits, r, a.ld, a.V);
  const int per = (row.vecs + cluster - 1) / cluster;
  const int v0 = min(rank * per, row.vecs), v1 = min(v0 + per, row.vecs);
  uint4 buf[kUnroll];
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) buf[u] = row.load(v0 + tid + u * nt, v1);
  int64_t y = -1;
  if (a.targets.p != nullptr) {
    y = load_id(a.targets, r);
    if (y < 0 || y >= a.V) {   // left out
      if (rank == 0) {
        if (tid == 0) {
          a.logprobs[r] = 0.f;
          a.entropy[r] = 0.f;
          a.stats[(size_t)r * 2] = a.stats[(size_t)r * 2 + 1] = 0.f;
        }
        for (int k = tid; k < K; k += nt) {
          a.top_logprobs[(size_t)r * K + k] = -inf_f();
          a.top_ids[(size_t)r * K + k] = -1;
        }
      }
      if (cluster > 1) cluster_wait();
      return;
    }
  }
  const float c2 = (float)(kLog2e / (double)a.temperature);
  const uint64_t c22 = pair(c2, c2);
  uint32_t* groups = reinterpret_cast<uint32_t*>(lists + (cluster > 1 ? cluster * K : 0));
  Sums t{-FLT_MAX, 0.f, 0.f};
  uint64_t l2[2] = {0, 0}, s2[2] = {0, 0};
#pragma unroll 1
  for (int s = 0; s < steps; ++s) {
    uint4 now[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) now[u] = buf[u];
    const int next = v0 + (s + 1) * kUnroll * nt + tid;
    if (s + 1 < steps) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) buf[u] = row.load(next + u * nt, v1);
    }
    uint32_t mw = Vec<T>::max_w(now[0]);
#pragma unroll
    for (int u = 1; u < kUnroll; ++u) mw = Elem<T>::max_w(mw, Vec<T>::max_w(now[u]));
    const float gm = Vec<T>::max_of(mw);
    if (TOP) groups[s * nt + tid] = order_key(gm);
    const float M = max_nan(t.m, gm);
    {
      const float d = fmaxf((t.m - M) * c2, kLeast), f = ex2(d);
      const uint64_t d2 = pair(d, d), f2 = pair(f, f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s2[i] = mul2(f2, fma2(l2[i], d2, s2[i]));
        l2[i] = mul2(l2[i], f2);
      }
      t.m = M;
    }
    const uint64_t nm = pair(-M, -M);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int i = 0; i < P; ++i) {
        float d0, d1;
        unpair(mul2(add2(Vec<T>::get(now[u], i), nm), c22), d0, d1);
        d0 = fmaxf(d0, kLeast);
        d1 = fmaxf(d1, kLeast);
        const uint64_t e = pair(ex2(d0), ex2(d1));
        l2[i & 1] = add2(l2[i & 1], e);
        s2[i & 1] = fma2(e, pair(d0, d1), s2[i & 1]);
      }
    }
  }
  {
    float x0, x1;
    unpair(add2(l2[0], l2[1]), x0, x1);
    t.l = x0 + x1;
    unpair(add2(s2[0], s2[1]), x0, x1);
    t.s = x0 + x1;
  }
  const float own_max = t.m;
  t = warp_join(t, c2);
  if (lane == 0) sh.part[warp] = t;
  if (TOP) {
    const uint32_t key = order_key(own_max);
    const uint32_t lo = __reduce_min_sync(0xffffffffu, key);
    if (lane == 0) {
      sh.wmin[warp] = lo;
      sh.wmax[warp] = order_key(t.m);
    }
    for (int i = tid; i < 80; i += nt) top.count[i] = 0;
    if (tid == 0) top.n = 0;
  }
  __syncthreads();
  if (cluster > 1) cluster_wait();   // every block of the cluster has started: its shared memory may be written
  if (warp == 0) {
    Sums b = lane < warps ? sh.part[lane] : Sums{-FLT_MAX, 0.f, 0.f};
    b = warp_join(b, c2);
    if (lane == 0) {
      if (cluster > 1) {
        store_to_cta(&sh.cta[rank][0], 0, b.m);
        store_to_cta(&sh.cta[rank][1], 0, b.l);
        store_to_cta(&sh.cta[rank][2], 0, b.s);
      } else {
        sh.cta[0][0] = b.m;
        sh.cta[0][1] = b.l;
        sh.cta[0][2] = b.s;
      }
    }
  }
  if (TOP) {
    uint32_t lo = sh.wmin[0], hi = sh.wmax[0];
    for (int w = 1; w < warps; ++w) {
      lo = min(lo, sh.wmin[w]);
      hi = max(hi, sh.wmax[w]);
    }
    const bool usable = !is_bad(key_value(hi)) && hi > kNegInfKey;   // else this block has no alternatives
    int n = 0;
    if (usable) {
      // the smallest of the threads' maxima has nt groups at or above it; with fewer than k, start below everything
      if (nt < K || lo <= kNegInfKey) lo = kNegInfKey + 1;
      auto share = [&](uint32_t bound) {
        int c = 0;
        for (int s = 0; s < steps; ++s) c += groups[s * nt + tid] >= bound;
        return c;
      };
      if (block_count(top, 79, share(lo)) >= K) lo = find_bound<uint32_t>(top, lo, hi + 1, Elem<T>::kStep, K, share);
      for (int s = 0; s < steps; ++s) {
        if (groups[s * nt + tid] < lo) continue;
#pragma unroll 1
        for (int u = 0; u < kUnroll; ++u) {
          const int i = v0 + (s * kUnroll + u) * nt + tid;
          const uint4 v = row.load(i, v1);
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int j = 0; j < Vec<T>::N; ++j) {
            const uint32_t key = order_key(to_f(e[j]));
            if (key >= lo) {
              const int at = atomicAdd(&top.n, 1);
              if (at < kCandidates) top.list[at] = alt_key(key, row.col(i) + j);
            }
          }
        }
      }
      __syncthreads();
      n = top.n;
      if (n > kCandidates) {
        __syncthreads();
        select_exactly<T>(top, row, v0, v1, K);
        n = top.n;
      }
    }
    rank_list(top, n, K);
    if (cluster > 1) {
      for (int k = tid; k < K; k += nt) store_to_cta(&lists[rank * K + k], 0, top.best[k]);
    }
  }
  if (cluster > 1) {
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
  } else {
    __syncthreads();
  }
  if (warp == 0) {
    Sums b = lane < cluster ? Sums{sh.cta[lane][0], sh.cta[lane][1], sh.cta[lane][2]} : Sums{-FLT_MAX, 0.f, 0.f};
    b = warp_join(b, c2);
    if (lane == 0) {
      const bool bad = is_bad(b.m), empty = !bad && b.l == 0.f;
      const double log_l = log((double)b.l);
      a.stats[(size_t)r * 2] = b.m;
      a.stats[(size_t)r * 2 + 1] = bad ? nan_f() : b.l;
      a.entropy[r] = bad ? nan_f() : (empty ? 0.f : (float)(log_l - kLn2 * (double)b.s / (double)b.l));
      if (y >= 0) {
        const double z = ((double)to_f(row.x[y]) - (double)b.m) / (double)a.temperature;
        a.logprobs[r] = bad ? nan_f() : (empty ? -inf_f() : (float)(z - log_l));
      }
      sh.m = b.m;
      sh.log_l_hi = (float)log_l;
      sh.log_l_lo = (float)(log_l - (double)sh.log_l_hi);
      sh.bad = bad;
    }
  }
  if (!TOP) return;
  if (cluster > 1) {
    // the cluster's lists: at most 8 x 128, in list once those below the k-th are gone
    const int all = cluster * K;
    clear_counts(top);
    auto share = [&](uint64_t bound) {
      int c = 0;
      for (int i = tid; i < all; i += nt) c += lists[i] >= bound;
      return c;
    };
    uint64_t lo = 1;
    if (block_count(top, 79, share(lo)) >= K) lo = find_bound<uint64_t>(top, lo, ~0ull, 1, K, share);
    if (tid == 0) top.n = 0;
    __syncthreads();
    for (int i = tid; i < all; i += nt)
      if (lists[i] >= lo) top.list[atomicAdd(&top.n, 1)] = lists[i];
    __syncthreads();
    rank_list(top, top.n, K);
  } else {
    __syncthreads();
  }
  const bool bad = sh.bad != 0;
  const double log_l = (double)sh.log_l_hi + (double)sh.log_l_lo;
  for (int k = tid; k < K; k += nt) {
    const uint64_t key = bad ? 0 : top.best[k];
    const double v = (double)key_value((uint32_t)(key >> 32));
    a.top_ids[(size_t)r * K + k] = key == 0 ? -1 : (int64_t)alt_col(key);
    a.top_logprobs[(size_t)r * K + k] =
        bad ? nan_f() : (key == 0 ? -inf_f() : (float)((v - (double)sh.m) / (double)a.temperature - log_l));
  }
}

// ------------------------------------------------------------------------------------------
// Writing a row of gradients: the output's rows may start at other addresses than the logits'
// ------------------------------------------------------------------------------------------
template <class T>
struct OutRow {
  T* p;
  bool vectors;   // its 16-byte boundaries are the logits'
  __device__ __forceinline__ OutRow(void* base, size_t row, int64_t ld, const Row<T>& in) : p(reinterpret_cast<T*>(base) + row * ld) {
    vectors = ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(in.x)) & 15) == 0;
  }
  __device__ __forceinline__ void store(const Row<T>& in, int i, const uint4& v) const {
    if (vectors && in.whole(i)) {
      *(reinterpret_cast<uint4*>(p - in.lead) + i) = v;
      return;
    }
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int k = 0; k < Vec<T>::N; ++k)
      if ((unsigned)(in.col(i) + k) < (unsigned)in.V) p[in.col(i) + k] = e[k];
  }
};
// One word of results from one or two values.
template <class T>
__device__ __forceinline__ void put_pair(uint4& v, int i, float a, float b) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&v);
  if constexpr (Elem<T>::kPerWord == 2) {
    w[i] = Elem<T>::narrow(a, b);
  } else {
    w[2 * i] = __float_as_uint(a);
    w[2 * i + 1] = __float_as_uint(b);
  }
}

// ------------------------------------------------------------------------------------------
// Gradients from a forward's statistics: one block a segment of a row. The columns named by the target and the
// alternatives (or by the teacher) get terms of their own: their logits are read before anything is written (the
// gradient may replace the logits), their results are written last.
// ------------------------------------------------------------------------------------------
constexpr int kGradVecs = 8;   // vectors of a thread, all in flight

struct EntryShared {
  int id[kHeadMaxTop + 1];
  float c[kHeadMaxTop + 1];
};

// f over all threads of the block. One barrier: slots may be written again after another one.
template <class F>
__device__ __forceinline__ float block_join(float v, float nothing, float* slots, F f) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  if (lane == 0) slots[warp] = v;
  __syncthreads();
  float r = nothing;
  for (int w = 0; w < warps; ++w) r = f(r, slots[w]);
  return r;
}
struct MaxF {
  __device__ float operator()(float a, float b) const { return max_nan(a, b); }
};
struct SumF {
  __device__ float operator()(float a, float b) const { return a + b; }
};

template <class T>
__global__ void __launch_bounds__(kThreads, 4) logprobs_bwd_kernel(LogprobsArgs a, int segments) {
  constexpr int P = Vec<T>::kPairs;
  __shared__ EntryShared sh;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int r = blockIdx.x / segments;
  const Row<T> row(a.logits, r, a.ld, a.V);
  const OutRow<T> out(a.d_logits, r, a.d_ld, row);
  const int v0 = (blockIdx.x % segments) * nt * kGradVecs, v1 = min(v0 + nt * kGradVecs, row.vecs);
  const float m = a.stats[(size_t)r * 2], l = a.stats[(size_t)r * 2 + 1];
  if (l == 0.f) {   // left out, or nothing is left
    for (int i = v0 + tid; i < v1; i += nt) out.store(row, i, make_uint4(0, 0, 0, 0));
    return;
  }
  uint4 buf[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) buf[u] = row.load(v0 + tid + u * nt, v1);
  // entries: the alternatives, then the target
  const int K = a.d_top != nullptr ? a.top_k : 0;
  const bool with_y = a.targets.p != nullptr && a.d_logprobs != nullptr;
  for (int k = tid; k <= K; k += nt) {
    int64_t id = -1;
    float c = 0.f;
    if (k < K) {
      id = a.top_ids[(size_t)r * K + k];
      if (id >= 0 && id < a.V) c = a.d_top[(size_t)r * K + k];
      else id = -1;
    } else if (with_y) {
      id = load_id(a.targets, r);
      if (id >= 0 && id < a.V) c = a.d_logprobs[r];
      else id = -1;
    }
    sh.id[k] = (int)id;
    sh.c[k] = c;
  }
  __syncthreads();
  float g = 0.f;
  for (int k = 0; k <= K; ++k) g += sh.c[k];
  const float it = 1.f / a.temperature, c2 = (float)(kLog2e / (double)a.temperature), inv_l = 1.f / l;
  const bool with_h = a.d_entropy != nullptr;
  // p (g + h (ln p + H)) = 2^d (A + B d)
  const float h = with_h ? a.d_entropy[r] : 0.f;
  const float B = -h * (float)kLn2 * inv_l;
  const float A = -inv_l * (with_h ? g + h * (float)((double)a.entropy[r] - log((double)l)) : g);
  auto dense = [&](float v) {
    const float d = fmaxf((v - m) * c2, kLeast);
    return ex2(d) * fmaf(B, d, A);
  };
  const int id = tid <= K ? sh.id[tid] : -1;     // a block has more threads than a row has entries
  const bool mine = id >= 0 && id >= row.col(v0) && id < row.col(v1);
  float own = 0.f;
  if (mine) {
    own = dense(to_f(row.x[id]));
    for (int k = 0; k <= K; ++k)
      if (sh.id[k] == id) own += sh.c[k];
  }
  __syncthreads();
  const uint64_t nm = pair(-m, -m), c22 = pair(c2, c2), B2 = pair(B * it, B * it), A2 = pair(A * it, A * it);
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int i = v0 + tid + u * nt;
    uint4 w;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      float d0, d1, x0, x1;
      unpair(mul2(add2(Vec<T>::get(buf[u], q), nm), c22), d0, d1);
      d0 = fmaxf(d0, kLeast);
      d1 = fmaxf(d1, kLeast);
      unpair(mul2(pair(ex2(d0), ex2(d1)), fma2(B2, pair(d0, d1), A2)), x0, x1);
      put_pair<T>(w, q, x0, x1);
    }
    if (i < v1) out.store(row, i, w);
  }
  __syncthreads();
  if (mine) from_f(own * it, out.p[id]);
}

// ------------------------------------------------------------------------------------------
// Distillation
// ------------------------------------------------------------------------------------------
struct TeacherShared {
  int id[kHeadMaxTop];
  float v[kHeadMaxTop];
  float red[3][kWarps];
};

// The teacher's entries of one row, one a thread (k = threadIdx.x < K).
struct Entry {
  int id;          // -1: absent
  bool first;      // the first with its token
  float q, q_all;  // its weight, and that of all entries with its token
  float x;         // the student's logit
  float v;         // log q up to the row's log_norm
};
struct Teacher {
  bool live;       // the row counts
  float log_norm;  // log q_k = v_k - log_norm
  float q_rest;    // what the bucket has left
};

// Loads the entries; a barrier. Every thread has the ids in sh.id and the values in sh.v afterwards.
__device__ __forceinline__ Entry load_entry(const DistillArgs& a, int r, TeacherShared& sh) {
  const int k = threadIdx.x;
  Entry e{-1, false, 0.f, 0.f, 0.f, -inf_f()};
  if (k < a.K) {
    const int64_t i = load_id(a.ids, (size_t)r * a.K + k);
    if (i >= 0 && i < a.V) {
      e.id = (int)i;
      e.v = load_value(a.values, a.value_type, (size_t)r * a.K + k);
    }
    sh.id[k] = e.id;
    sh.v[k] = e.v;
  }
  __syncthreads();
  return e;
}
// Weights; two barriers.
__device__ __forceinline__ Teacher weigh(const DistillArgs& a, TeacherShared& sh, Entry& e) {
  Teacher t;
  const float vm = block_join(e.v, -inf_f(), sh.red[0], MaxF());
  const bool any = __syncthreads_or(e.id >= 0);
  t.live = any && (a.bucket || vm != -inf_f());
  const float base = a.bucket ? 0.f : vm;
  const float w = e.id >= 0 ? ex2((e.v - base) * (float)kLog2e) : 0.f;
  const float total = block_join(w, 0.f, sh.red[1], SumF());
  const float norm = a.bucket ? 1.f : 1.f / total;
  t.log_norm = a.bucket ? 0.f : (float)((double)vm + log((double)total));
  t.q_rest = a.bucket ? fmaxf(0.f, 1.f - total) : 0.f;
  e.q = w * norm;
  e.first = e.id >= 0;
  if (e.id >= 0) {
    for (int k = 0; k < a.K; ++k) {
      if (sh.id[k] != e.id) continue;
      if (k < (int)threadIdx.x) e.first = false;
      e.q_all += ex2((sh.v[k] - base) * (float)kLog2e) * norm;
    }
  }
  return t;
}

// Loss (and gradient). The columns of the teacher's tokens are kept apart: the sum over all others is taken relative
// to their own maximum, so that the mass outside keeps its digits when the teacher's tokens have nearly all of it.
// stats = (maximum outside, coefficient of 2^d outside, maximum, 1 / l); the last is -1 for a row that is left out.
//
// The blocks of a cluster share a row. HELD: a thread keeps its vectors in registers from the maximum to the gradient, so
// the logits are read once; otherwise (more columns than the cluster's registers hold) each step reads them again.
template <class T, int NV, bool HELD, bool WRITE>
__global__ void __launch_bounds__(kThreads, NV >= 8 ? 4 : 5) distill_kernel(DistillArgs a, int cluster) {
  constexpr int P = Vec<T>::kPairs, N = Vec<T>::N;
  extern __shared__ uint32_t marks[];            // a byte for each vector of the block: columns of the teacher's tokens
  __shared__ TeacherShared sh;
  __shared__ float red[4][kWarps];
  __shared__ float cta[kMaxCluster][2];
  __shared__ double red64[kWarps][2];
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  const int r = blockIdx.x / cluster, rank = blockIdx.x % cluster;
  if (cluster > 1) cluster_arrive();
  const Row<T> row(a.logits, r, a.ld, a.V);
  const int chunk = nt * NV;
  int per = (row.vecs + cluster - 1) / cluster;
  const int chunks = HELD ? 1 : (per + chunk - 1) / chunk;
  const int v0 = min(rank * per, row.vecs), v1 = min(v0 + per, row.vecs);
  for (int i = tid; i < chunks * chunk / 4; i += nt) marks[i] = 0;
  uint4 buf[NV];
  auto fetch = [&](int c) {
#pragma unroll
    for (int u = 0; u < NV; ++u) buf[u] = row.load(v0 + c * chunk + tid + u * nt, v1);
  };
  Entry e = load_entry(a, r, sh);       // its barrier: marks are clear
  if (HELD) fetch(0);
  if (e.id >= 0) {
    e.x = to_f(row.x[e.id]);
    const int v = (e.id + row.lead) / N, j = (e.id + row.lead) % N;
    if (v >= v0 && v < v1) {
      const int at = v - v0, c = at / chunk, in = at % chunk;
      const int byte = c * chunk + (in % nt) * NV + in / nt;    // a thread's bytes lie side by side
      atomicOr(&marks[byte >> 2], 1u << ((byte & 3) * 8 + j));
    }
  }
  const Teacher t = weigh(a, sh, e);    // its barriers: marks are set
  OutRow<T> out(WRITE ? a.d_logits : const_cast<void*>(a.logits), r, WRITE ? a.d_ld : a.ld, row);
  if (!t.live) {
    if (rank == 0 && tid == 0) {
      a.loss[r] = 0.f;
      if (!WRITE) reinterpret_cast<float4*>(a.stats)[r] = make_float4(0.f, 0.f, 0.f, -1.f);
    }
    if (WRITE)
      for (int i = v0 + tid; i < v1; i += nt) out.store(row, i, make_uint4(0, 0, 0, 0));
    if (cluster > 1) cluster_wait();
    return;
  }
  auto drop_marked = [&](int c) {
    const uint8_t* mine = reinterpret_cast<const uint8_t*>(marks) + c * chunk + tid * NV;
    uint32_t any = 0;
#pragma unroll
    for (int u = 0; u < NV; ++u) any |= mine[u];
    if (any) {
#pragma unroll
      for (int u = 0; u < NV; ++u) Vec<T>::drop(buf[u], mine[u]);
    }
  };
  // maxima: of what is outside (of this block's part), and of the teacher's tokens
  float mr = -FLT_MAX;
  for (int c = 0; c < chunks; ++c) {
    if (!HELD) fetch(c);
    drop_marked(c);
    uint32_t mw = Vec<T>::max_w(buf[0]);
#pragma unroll
    for (int u = 1; u < NV; ++u) mw = Elem<T>::max_w(mw, Vec<T>::max_w(buf[u]));
    mr = max_nan(mr, Vec<T>::max_of(mw));
  }
  mr = block_join(mr, -FLT_MAX, red[0], MaxF());
  const float mt = block_join(e.id >= 0 ? e.x : -inf_f(), -FLT_MAX, red[1], MaxF());
  const float c2 = (float)(kLog2e / (double)a.temperature);
  const uint64_t c22 = pair(c2, c2);
  float lr = 0.f;
  {
    const uint64_t nm = pair(-mr, -mr);
    uint64_t l2[2] = {0, 0};
    for (int c = 0; c < chunks; ++c) {
      if (!HELD) {
        fetch(c);
        drop_marked(c);
      }
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int q = 0; q < P; ++q) {
          float d0, d1;
          unpair(mul2(add2(Vec<T>::get(buf[u], q), nm), c22), d0, d1);
          l2[q & 1] = add2(l2[q & 1], pair(ex2(d0), ex2(d1)));
        }
    }
    float x0, x1;
    unpair(add2(l2[0], l2[1]), x0, x1);
    lr = x0 + x1;
  }
  lr = block_join(lr, 0.f, red[2], SumF());
  const float lt = block_join(e.first && e.x != -inf_f() ? ex2((e.x - mt) * c2) : 0.f, 0.f, red[3], SumF());
  // sum of q_k (log q_k - (x_k - mt) / t), in 64 bits: its terms are larger than what is left of them
  double terms = 0., weight = e.q;
  if (e.id >= 0 && e.q != 0.f) {
    const double z = e.x == -inf_f() ? -(double)inf_f() : ((double)e.x - (double)mt) / (double)a.temperature;
    terms = (double)e.q * ((double)e.v - (double)t.log_norm - z);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    terms += __shfl_xor_sync(0xffffffffu, terms, o);
    weight += __shfl_xor_sync(0xffffffffu, weight, o);
  }
  if (lane == 0) {
    red64[warp][0] = terms;
    red64[warp][1] = weight;
  }
  if (cluster > 1) {
    __syncthreads();
    cluster_wait();        // every block has started
    if (tid < cluster) {
      store_to_cta(&cta[rank][0], tid, mr);
      store_to_cta(&cta[rank][1], tid, lr);
    }
    cluster_arrive();
    cluster_wait();
    float M = -FLT_MAX;
    for (int c = 0; c < cluster; ++c) M = max_nan(M, cta[c][0]);
    lr = 0.f;
    for (int c = 0; c < cluster; ++c) lr += cta[c][1] * ex2(fmaxf((cta[c][0] - M) * c2, kLeast));
    mr = M;
  } else {
    __syncthreads();
  }
  const float m = max_nan(mr, mt);
  const float share = ex2((mr - m) * c2);
  const float l = lt * ex2((mt - m) * c2) + lr * share;
  const bool bad = is_bad(m);
  const float inv_l = bad ? nan_f() : (l == 0.f ? 0.f : 1.f / l);
  const float coef = bad ? nan_f() : (lr == 0.f ? 0.f : share * inv_l - t.q_rest / lr);
  if (rank == 0 && tid == 0) {
    double loss = 0., q = 0.;
    for (int w = 0; w < warps; ++w) {
      loss += red64[w][0];
      q += red64[w][1];
    }
    const double log_l = log((double)l);
    // + the sum of q_k times the rest of -log p_k; a student with nothing has infinite terms already
    if (l != 0.f) loss += q * (log_l - ((double)mt - (double)m) / (double)a.temperature);
    if (t.q_rest > 0.f && lr != 0.f) {
      const double lp = ((double)mr - (double)m) / (double)a.temperature + log((double)lr) - log_l;
      loss += (double)t.q_rest * (log((double)t.q_rest) - lp);
    }
    a.loss[r] = bad ? nan_f() : (float)loss;
    if (!WRITE) reinterpret_cast<float4*>(a.stats)[r] = make_float4(mr, coef, m, inv_l);
  }
  if (!WRITE) return;
  const float w = a.grad_scale / a.temperature;
  const uint64_t nm = pair(-mr, -mr), w2 = pair(w * coef, w * coef);
  for (int c = 0; c < chunks; ++c) {
    if (!HELD) {
      fetch(c);
      drop_marked(c);
    }
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i = v0 + c * chunk + tid + u * nt;
      uint4 g;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        float d0, d1, x0, x1;
        unpair(mul2(add2(Vec<T>::get(buf[u], q), nm), c22), d0, d1);
        unpair(mul2(pair(ex2(d0), ex2(d1)), w2), x0, x1);
        put_pair<T>(g, q, x0, x1);
      }
      if (i < v1) out.store(row, i, g);
    }
  }
  __syncthreads();
  if (e.first) {
    const int v = (e.id + row.lead) / N;
    if (v >= v0 && v < v1) {
      const float p = inv_l * (e.x == -inf_f() ? 0.f : ex2((e.x - m) * c2));
      from_f(w * (p - e.q_all), out.p[e.id]);
    }
  }
}

// Gradient from the forward's statistics, one block a segment of a row.
template <class T>
__global__ void __launch_bounds__(kThreads, 4) distill_bwd_kernel(DistillArgs a, int segments) {
  constexpr int P = Vec<T>::kPairs, N = Vec<T>::N;
  __shared__ TeacherShared sh;
  const int tid = threadIdx.x, nt = blockDim.x;
  const int r = blockIdx.x / segments;
  const Row<T> row(a.logits, r, a.ld, a.V);
  const OutRow<T> out(a.d_logits, r, a.d_ld, row);
  const int v0 = (blockIdx.x % segments) * nt * kGradVecs, v1 = min(v0 + nt * kGradVecs, row.vecs);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[r];
  if (st.w < 0.f) {
    for (int i = v0 + tid; i < v1; i += nt) out.store(row, i, make_uint4(0, 0, 0, 0));
    return;
  }
  uint4 buf[kGradVecs];
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) buf[u] = row.load(v0 + tid + u * nt, v1);
  Entry e = load_entry(a, r, sh);
  weigh(a, sh, e);
  const float mr = st.x, coef = st.y, m = st.z, inv_l = st.w;
  const float c2 = (float)(kLog2e / (double)a.temperature), w = a.d_loss[r] / a.temperature;
  bool mine = false;
  float own = 0.f;
  if (e.first) {
    const int v = (e.id + row.lead) / N;
    if (v >= v0 && v < v1) {
      mine = true;
      e.x = to_f(row.x[e.id]);
      own = w * (inv_l * (e.x == -inf_f() ? 0.f : ex2((e.x - m) * c2)) - e.q_all);
    }
  }
  __syncthreads();
  const uint64_t nm = pair(-mr, -mr), c22 = pair(c2, c2), w2 = pair(w * coef, w * coef);
#pragma unroll
  for (int u = 0; u < kGradVecs; ++u) {
    const int i = v0 + tid + u * nt;
    uint4 g;
#pragma unroll
    for (int q = 0; q < P; ++q) {
      float d0, d1, x0, x1;
      unpair(mul2(add2(Vec<T>::get(buf[u], q), nm), c22), d0, d1);
      // the teacher's tokens may lie above the maximum of the others; they are written below
      unpair(mul2(pair(ex2(fminf(d0, 0.f)), ex2(fminf(d1, 0.f))), w2), x0, x1);
      put_pair<T>(g, q, x0, x1);
    }
    if (i < v1) out.store(row, i, g);
  }
  __syncthreads();
  if (mine) from_f(own, out.p[e.id]);
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
int threads_for(int vecs, int least) {
  const int n = ((vecs > least ? vecs : least) + 31) / 32 * 32;
  return n < kThreads ? n : kThreads;
}
template <class... P, class... A>
void launch(void (*kernel)(P...), int rows, int blocks_a_row, bool cluster, int threads, int smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)rows * (unsigned)blocks_a_row);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks_a_row;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster && blocks_a_row > 1 ? 1 : 0;
  if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  cudaLaunchKernelEx(&cfg, kernel, args...);
}

template <class T>
void launch_fwd(const LogprobsArgs& a) {
  const int vecs = most_vecs<T>(a.logits, a.ld, a.rows, a.V);
  const int threads = threads_for(vecs, 32);
  // Blocks a row: one fills the machine's memory pipes when there are four blocks for each SM; fewer rows are split as
  // long as a block keeps a vector for each thread. A block's group maxima take at most 64 KB.
  int cluster = 1;
  while (cluster < kMaxCluster && (int64_t)a.rows * cluster * 2 <= 4 * a.sm_count && vecs / (cluster * 2) >= threads) cluster *= 2;
  while (cluster < kMaxCluster && vecs / cluster > 64 * threads * kUnroll) cluster *= 2;
  const int per = (vecs + cluster - 1) / cluster;
  const int steps = (per + threads * kUnroll - 1) / (threads * kUnroll);
  if (a.top_k > 0) {
    const int smem = (int)sizeof(TopShared) + (cluster > 1 ? cluster * a.top_k * 8 : 0) + steps * threads * 4;
    launch(logprobs_fwd_kernel<T, true>, a.rows, cluster, true, threads, smem, a.stream, a, cluster, steps);
  } else {
    launch(logprobs_fwd_kernel<T, false>, a.rows, cluster, true, threads, 0, a.stream, a, cluster, steps);
  }
}

template <class T>
void launch_bwd(const LogprobsArgs& a) {
  const int vecs = most_vecs<T>(a.logits, a.ld, a.rows, a.V);
  const int threads = threads_for(vecs, (a.d_top != nullptr ? a.top_k : 0) + 1);
  const int segments = (vecs + threads * kGradVecs - 1) / (threads * kGradVecs);
  launch(logprobs_bwd_kernel<T>, a.rows, segments, false, threads, 0, a.stream, a, segments);
}

template <class T, bool WRITE, int NV, bool HELD>
void launch_distill_as(const DistillArgs& a, int vecs, int threads, int cluster) {
  const int per = (vecs + cluster - 1) / cluster, chunk = threads * NV;
  const int smem = (per + chunk - 1) / chunk * chunk;
  launch(distill_kernel<T, NV, HELD, WRITE>, a.rows, cluster, true, threads, smem, a.stream, a, cluster);
}
template <class T, bool WRITE>
void launch_distill(const DistillArgs& a) {
  const int vecs = most_vecs<T>(a.logits, a.ld, a.rows, a.V);
  const int threads = threads_for(vecs, a.K);
  // Blocks a row: as many as hold it in registers, eight vectors a thread; more for few rows.
  int cluster = 1;
  while (cluster < kMaxCluster && vecs > cluster * threads * 8) cluster *= 2;
  while (cluster < kMaxCluster && (int64_t)a.rows * cluster * 2 <= 4 * a.sm_count && vecs / (cluster * 2) >= threads) cluster *= 2;
  const int per = (vecs + cluster - 1) / cluster;
  if (per <= threads) launch_distill_as<T, WRITE, 1, true>(a, vecs, threads, cluster);
  else if (per <= threads * 2) launch_distill_as<T, WRITE, 2, true>(a, vecs, threads, cluster);
  else if (per <= threads * 4) launch_distill_as<T, WRITE, 4, true>(a, vecs, threads, cluster);
  else if (per <= threads * 8) launch_distill_as<T, WRITE, 8, true>(a, vecs, threads, cluster);
  else launch_distill_as<T, WRITE, 8, false>(a, vecs, threads, cluster);
}

}  // namespace

void launch_token_logprobs_fwd(const LogprobsArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { launch_fwd<decltype(t)>(a); });
}
void launch_token_logprobs_bwd(const LogprobsArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { launch_bwd<decltype(t)>(a); });
}
void launch_distill_fwd(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { launch_distill<decltype(t), false>(a); });
}
void launch_distill_bwd(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) {
    using T = decltype(t);
    const int vecs = most_vecs<T>(a.logits, a.ld, a.rows, a.V);
    const int threads = threads_for(vecs, a.K);
    const int segments = (vecs + threads * kGradVecs - 1) / (threads * kGradVecs);
    launch(distill_bwd_kernel<T>, a.rows, segments, false, threads, 0, a.stream, a, segments);
  });
}
void launch_distill_fwd_bwd(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { launch_distill<decltype(t), true>(a); });
}

}  // namespace zx
