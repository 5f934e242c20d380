// Token log-probabilities: for logits x [rows, V], z = x / temperature, lse = log sum exp z, p = exp(z - lse),
//   forward:   z_y - lse of a given token y, the entropy H = -sum p (z - lse), the k most likely tokens;
//   backward:  d/dx_j = (1 / temperature) [ g ([j = y] - p_j) - h p_j (z_j - lse + H) + sum_k c_k ([j = i_k] - p_j) ].
// Both are bound by the bytes of the logits, read once each way. With l = sum 2^d, s = sum 2^d d (d = rel2, rows.cuh):
// z_j - lse = ln 2 (d_j - log2 l), H = ln 2 (log2 l - s / l). d of the maximum is not 0 but the rounding of its reference (2^-5 at
// most), so both terms of H may be that far from their sign, and where one token has all the mass they cancel: H and z_j - lse
// are off by what l and s are, relatively (2^-22 and more with V), and are held at 0, which they would pass. (maximum, l) is what
// the backward needs. Sums are held in 32 bits, the few scalars of a row are put together in 64.
//
// Measured on a B200 that copies 6557 GB/s: forward 4096 x 128256 bf16 160 us (6.6 TB/s), with 20 alternatives 199, 64
// 218, 128 242; one row 4.7 us, with 20 alternatives 7.9 (launch and the search's chain of barriers); 64 x 128256 fp32
// 10.3 us (3.2 TB/s: a cluster's start and end are as long as its slice), with 20 alternatives 15.4. Backward 2048 x 128256
// bf16 160 us (6.6 TB/s), 4096 rows with 64 alternatives 336.
#include <algorithm>
#include "rows.cuh"

namespace zx {

namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
// Vectors of a thread whose maximum is kept (a group). Eight: 4096 x 128256, 64 alternatives, 240 us instead of 219 (twice as
// many logits are looked at again).
constexpr int kUnroll = 4;
constexpr int kGradVecs = 8;    // vectors of a thread in the backward, all in flight

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

// (maximum m, l = sum 2^rel2, s = sum 2^rel2 rel2)
struct Sums {
  float m, l, s;
};
__device__ __forceinline__ void move_to(Sums& a, float M, float c2) {
  const float d = gap2(a.m, M, c2), f = ex2(d);
  a.s = f * (a.s + a.l * d);
  a.l *= f;
  a.m = M;
}
__device__ __forceinline__ Sums warp_join(Sums a, float c2) {
  move_to(a, warp_max_nan(a.m), c2);
  a.l = warp_sum(a.l);
  a.s = warp_sum(a.s);
  return a;
}

// ------------------------------------------------------------------------------------------
// The k best of a row, in a block
// ------------------------------------------------------------------------------------------
constexpr int kCandidates = 1024;

static_assert(kCandidates >= kMaxCluster * kHeadMaxTop, "the lists of a cluster");
constexpr int kGroups = 512;    // groups whose vectors are looked at again

struct TopShared {
  uint64_t list[kCandidates + 32];
  uint64_t best[kHeadMaxTop];
  uint32_t hist[256];
  int group[kGroups];     // step and thread
  uint32_t lo;
  int n, count, above, groups;
  int warp[kWarps];
};

// Descending over the lanes of a warp (bitonic).
template <class Key>
__device__ __forceinline__ Key warp_sort(Key key) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size *= 2) {
#pragma unroll
    for (int o = size / 2; o > 0; o /= 2) {
      const Key other = __shfl_xor_sync(0xffffffffu, key, o);
      const bool larger = ((lane & o) == 0) == ((lane & size) == 0 || size == 32);
      key = larger == (other > key) ? other : key;
    }
  }
  return key;
}

// A bound with at least k of the block's group maxima at or above it, and few more: a histogram over [lo, hi] (which
// holds the k-th largest), and again over the bin that holds it while that is crowded. groups: [steps][threads].
__device__ __forceinline__ uint32_t find_bound(TopShared& sh, const uint32_t* groups, int steps, uint32_t lo, uint32_t hi, int k) {
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31;
  int above = 0;
#pragma unroll 1
  for (int pass = 0; pass < 4; ++pass) {
    const uint32_t span = hi - lo;
    const int shift = span < 256u ? 0 : 24 - __clz(span);
    for (int i = tid; i < 256; i += nt) sh.hist[i] = 0;
    __syncthreads();
    for (int s = 0; s < steps; ++s) {
      const uint32_t key = groups[s * nt + tid];
      if (key >= lo && key <= hi) atomicAdd(&sh.hist[(key - lo) >> shift], 1u);
    }
    __syncthreads();
    if (tid < 32) {
      int c[8], mine = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        c[i] = (int)sh.hist[lane * 8 + i];
        mine += c[i];
      }
      int from = mine;      // in this lane's bins and those above
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_down_sync(0xffffffffu, from, o);
        if (lane + o < 32) from += up;
      }
      const uint32_t enough = __ballot_sync(0xffffffffu, above + from >= k);
      if (lane == 0 && enough == 0) sh.count = -1;
      if (enough != 0 && lane == 31 - __clz(enough)) {     // the last lane with enough
        int over = above + from - mine, b = 7;
        for (; b > 0 && over + c[b] < k; --b) over += c[b];
        sh.lo = lo + ((uint32_t)(lane * 8 + b) << shift);
        sh.count = over + c[b];
        sh.above = over;
      }
    }
    __syncthreads();
    if (sh.count < 0) return lo;      // fewer than k: all
    lo = sh.lo;
    if (shift == 0 || sh.count <= k + k / 2 + 16) return lo;
    hi = min(hi, lo + ((1u << shift) - 1));
    above = sh.above;
  }
  return lo;
}

__device__ __forceinline__ void first_threads_sync(int n) { asm volatile("bar.sync 1, %0;" ::"r"(n) : "memory"); }

// How many of the 32 keys at run (descending) are above key.
__device__ __forceinline__ int above_in_run(const uint64_t* run, uint64_t key) {
  int c = 0;
#pragma unroll
  for (int step = 16; step > 0; step /= 2)
    if (run[c + step - 1] > key) c += step;
  return c + (run[c] > key ? 1 : 0);
}
// best[0 .. k) = the k largest of list[0 .. n), in order (0 where there are fewer). Needs a barrier before, ends with one.
// Up to 128 members: each counts those above it, with the help of neighbouring lanes (one row, 20 alternatives: 8.0 us with
// this, 9.0 with runs alone; for more members the runs take fewer steps). More: runs of 32 are sorted, each by
// a warp; a member's place is its own in the run plus, in each other run, the number above it.
// Called by the first nt threads.
__device__ __forceinline__ void rank_list(TopShared& sh, int n, int k, int nt) {
  const int tid = threadIdx.x, runs = (n + 31) / 32;
  for (int i = n + tid; i < k; i += nt) sh.best[i] = 0;
  if (n <= 128) {
    const int shift = min(5, max(0, 31 - __clz(nt / max(n, 1)))), lanes = 1 << shift;      // for one member
    const int part = tid & (lanes - 1);
    for (int first = 0; first < n; first += nt >> shift) {
      const int at = first + (tid >> shift);
      const uint64_t mine = at < n ? sh.list[at] : ~0ull;
      int r = 0;
#pragma unroll 4
      for (int i = part; i < n; i += lanes) r += sh.list[i] > mine;
      for (int o = lanes / 2; o > 0; o /= 2) r += __shfl_xor_sync(0xffffffffu, r, o);
      if (part == 0 && at < n && r < k) sh.best[r] = mine;
    }
    first_threads_sync(nt);
    return;
  }
  for (int i = tid; i < runs * 32; i += nt) sh.list[i] = warp_sort(i < n ? sh.list[i] : (uint64_t)0);
  if (tid < 32) sh.list[runs * 32 + tid] = 0;      // an empty run behind the last
  first_threads_sync(nt);
  for (int i = tid; i < runs * 32; i += nt) {
    const uint64_t mine = sh.list[i];
    int r = i & 31;
    if (mine == 0 || r >= k) continue;
    r = 0;      // (the own run gives the own place)
    for (int c = 0; c < runs; c += 4) {       // four at once: the searches are chains of loads
#pragma unroll
      for (int b = 0; b < 4; ++b) r += above_in_run(&sh.list[min(c + b, runs) * 32], mine);
    }
    if (r < k) sh.best[r] = mine;
  }
  first_threads_sync(nt);
}

// Where a thread's `mine` entries start in a list of *n so far: one atomic a warp.
__device__ __forceinline__ int take_places(int* n, int mine) {
  const int lane = threadIdx.x & 31;
  int upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, upto, o);
    if (lane >= o) upto += up;
  }
  int first = 0;
  if (lane == 31 && upto > 0) first = atomicAdd(n, upto);
  return __shfl_sync(0xffffffffu, first, 31) + upto - mine;
}

// The same of `lists` sorted lists of k each (of the blocks of a cluster). Called by the first nt threads.
__device__ __forceinline__ void merge_lists(TopShared& sh, const uint64_t* list, int lists, int k, int nt) {
  // The k-th is not below the smallest of the lists' members number ceil(k / lists), nor below any list's last.
  const int q = (k + lists - 1) / lists, lane = threadIdx.x & 31;
  const bool one = lane < lists;
  const uint32_t least = __reduce_min_sync(0xffffffffu, one ? (uint32_t)(list[lane * k + q - 1] >> 32) : 0xffffffffu);
  const uint32_t last = __reduce_max_sync(0xffffffffu, one ? (uint32_t)(list[lane * k + k - 1] >> 32) : 0);
  const uint64_t lo = max((uint64_t)max(least, last) << 32, (uint64_t)1);
  if (threadIdx.x == 0) sh.n = 0;
  first_threads_sync(nt);
  for (int i = threadIdx.x; i - (int)(threadIdx.x & 31) < lists * k; i += nt) {   // whole warps
    const uint64_t key = i < lists * k ? list[i] : 0;
    const int at = take_places(&sh.n, key >= lo);
    if (key >= lo) sh.list[at] = key;
  }
  first_threads_sync(nt);
  rank_list(sh, sh.n, k, nt);
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
    for (int i = v0 + tid; i - lane < v1; i += blockDim.x) {   // whole warps
      const uint4 v = row.load(i, v1);
      const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const uint32_t key = order_key(to_f(e[j]));
        const bool in = key > kNegInfKey && (key & mask) == prefix;
        const uint32_t digit = in ? (key >> shift & 255u) : 256u;
        const uint32_t same = __match_any_sync(0xffffffffu, digit);
        if (in && (int)__ffs(same) - 1 == lane) atomicAdd(&sh.hist[digit], (uint32_t)__popc(same));
      }
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255, above = 0;
      for (; d > 0; --d) {
        if (above + (int)sh.hist[d] >= need) break;
        above += (int)sh.hist[d];
      }
      sh.lo = (uint32_t)d;
      sh.above = above;
    }
    __syncthreads();
    prefix |= sh.lo << shift;
    mask |= 255u << shift;
    need -= sh.above;
    __syncthreads();
  }
  if (prefix <= kNegInfKey) prefix = kNegInfKey;   // fewer than k: all that there are are above it
  if (tid == 0) sh.n = 0;
  int ties = 0;   // of those before the vectors at hand
  __syncthreads();
  for (int base = v0; base < v1; base += blockDim.x) {
    const int i = base + tid;
    const uint4 v = row.load(i, v1);
    const T* e = reinterpret_cast<const T*>(&v);
    int equal = 0;
#pragma unroll
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
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const uint32_t key = order_key(to_f(e[j]));
      if (key != prefix || equal == 0) continue;
      if (place < need) sh.list[atomicAdd(&sh.n, 1)] = alt_key(key, row.col(i) + j);
      ++place;
    }
    ties = all;
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------------
// Forward: one pass over the row, by a block or by a cluster of them
// ------------------------------------------------------------------------------------------
struct FwdShared {
  Sums part[kWarps];
  float cta[kMaxCluster][3];
  float m;
  double log_l;
  uint32_t least[4][kWarps], most[kWarps];
  __align__(16) uint32_t own[kThreads];
};

// One group of vectors into the running sums (l and s as pairs).
template <class T, bool Far, int U>
__device__ __forceinline__ void add_group(const uint4 (&v)[U], float M, float c2, uint64_t (&l2)[2], uint64_t (&s2)[2]) {
  const Rel2<Far> rel(M, c2);
  // -inf stays out of the entropy: in bf16 as a large finite number (two at once), which M is far above
  constexpr bool kClampWords = std::is_same<T, __nv_bfloat16>::value && !Far;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    uint4 w = v[u];
    if (kClampWords) {
      constexpr uint32_t kLow = 0xf149f149u;     // -9.98e29 (|M| is below 1e11 here)
      w.x = Elem<T>::max_w(w.x, kLow);
      w.y = Elem<T>::max_w(w.y, kLow);
      w.z = Elem<T>::max_w(w.z, kLow);
      w.w = Elem<T>::max_w(w.w, kLow);
    }
#pragma unroll
    for (int i = 0; i < Vec<T>::kPairs; ++i) {
      uint64_t d = rel(Vec<T>::get(w, i));
      float d0, d1;
      unpair(d, d0, d1);
      if (!kClampWords) {
        d0 = fmaxf(d0, kLeast);
        d1 = fmaxf(d1, kLeast);
        d = pair(d0, d1);
      }
      const uint64_t e = pair(ex2(d0), ex2(d1));
      l2[i & 1] = add2(l2[i & 1], e);
      s2[i & 1] = fma2(e, d, s2[i & 1]);
    }
  }
}

// A block walks its slice of the row once, with a running maximum and sums that move to a larger maximum when one comes.
//
// TOP: a thread keeps the maximum of each of its groups (kUnroll vectors) in shared memory. Any bound with k group maxima
// at or above it bounds the k-th largest logit from below, so only those groups are read again, from the L2 cache mostly.
// The first bound comes from the threads' maxima: 2^j warps with ceil(k / 2^j) threads each, the best over j. Where it lets
// more than 2 k + 32 groups pass, a histogram of the group maxima gives a better one (always: 4096 x 128256, one
// alternative, 206 us instead of 191; never: 999 x 50257 fp16, 128 alternatives, 79 instead of 45); where that does not
// help either (ties, large logits side by side), the k are selected by their digits from all of the row.
// What the search costs is its chain of barriers and reads, in which a block asks for little: 7 us of a row's 29 at 4096 x
// 128256. Of the 13,800 clocks that one row with 20 alternatives takes, 3500 are the scan, 1300 sums and bound, 550 the list
// of groups, 2000 the second look, 1200 the order, 1200 the exchange in the cluster, 2500 the merge. Copies into shared
// memory ahead of their use (a ring for each warp) made it 242 us instead of 219, larger steps 240, the next row's start in the
// L2 cache 227.
template <class T, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) logprobs_fwd_kernel(LogprobsArgs a, int cluster, int steps) {
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
  row.load_group(buf, v0, v0 + tid, nt, v1);
  int64_t y = -1;
  if (a.targets.p != nullptr) {
    y = load_id(a.targets, r);
    if (y < 0 || y >= a.V) {   // left out
      if (rank == 0) {
        if (tid == 0) {
          a.logprobs[r] = 0.f;
          a.entropy[r] = 0.f;
          if (a.stats != nullptr) a.stats[(size_t)r * 2] = a.stats[(size_t)r * 2 + 1] = 0.f;
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
  float xy = 0.f;
  if (y >= 0 && warp == warps - 1) xy = to_f(row.x[y]);
  const float c2 = scale2(a.temperature);
  uint32_t* groups = reinterpret_cast<uint32_t*>(lists + (cluster > 1 ? cluster * K : 0));
  Sums t{-FLT_MAX, 0.f, 0.f};
  uint64_t l2[2] = {0, 0}, s2[2] = {0, 0};
  auto add = [&](const auto& v, int s) {
    constexpr int U = sizeof(v) / sizeof(v[0]);
    uint32_t mw = Vec<T>::max_w(v[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) mw = Elem<T>::max_w(mw, Vec<T>::max_w(v[u]));
    const float gm = Vec<T>::max_of(mw);
    if (TOP) groups[s * nt + tid] = order_key(gm);
    const float M = max_nan(t.m, gm), R = ref2(M, c2);
    auto move = [&](float d) {
      const float f = ex2(d);
      const uint64_t d2 = pair(d, d), f2 = pair(f, f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s2[i] = mul2(f2, fma2(l2[i], d2, s2[i]));
        l2[i] = mul2(l2[i], f2);
      }
      t.m = M;
    };
    if (plain_gap(R)) {
      move(gap2_plain(t.m, R, c2));
      add_group<T, false>(v, M, c2, l2, s2);
    } else {
      move(gap2_far(t.m, M, c2));
      if (is_far(M, c2)) add_group<T, true>(v, M, c2, l2, s2);
      else add_group<T, false>(v, M, c2, l2, s2);
    }
  };
  if (TOP) {
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
      uint4 now[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) now[u] = buf[u];
      if (s + 1 < steps) {
        const int next = v0 + (s + 1) * kUnroll * nt;
        row.load_group(buf, next, next + tid, nt, v1);
      }
      add(now, s);
    }
  } else {
    // eight at a time, without a second buffer: 187 against 192 us for 4096 x 128256 bf16, time after time
    add(buf, 0);
#pragma unroll 1
    for (int i = v0 + kUnroll * nt; i < v1; i += 2 * kUnroll * nt) {
      uint4 now[2 * kUnroll];
      row.load_group(now, i, i + tid, nt, v1);
      add(now, 0);
    }
  }
  {
    float x0, x1;
    unpair(add2(l2[0], l2[1]), x0, x1);
    t.l = x0 + x1;
    unpair(add2(s2[0], s2[1]), x0, x1);
    t.s = x0 + x1;
  }
  const uint32_t own = order_key(t.m);
  t = warp_join(t, c2);
  if (lane == 0) sh.part[warp] = t;
  if (TOP) {
    // What ceil(K / 2^j) of the warp's threads reach: the smallest that fewer are above.
    sh.own[tid] = own;
    __syncwarp();
    int above = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 o = reinterpret_cast<const uint4*>(&sh.own[warp * 32])[i];
      above += (o.x > own) + (o.y > own) + (o.z > own) + (o.w > own);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int q = (K + (1 << j) - 1) >> j;
      const uint32_t least = __reduce_min_sync(0xffffffffu, above < q ? own : 0xffffffffu);
      if (lane == 0) sh.least[j][warp] = q <= 32 ? least : 0;
    }
    if (lane == 0) {
      sh.most[warp] = order_key(t.m);
    }
    if (tid == 0) top.n = top.groups = 0;
  }
  __syncthreads();
  // What the row as a whole gives, once its sums are in one warp.
  auto tell = [&](const Sums& b) {
    if (lane != 0) return;
    const bool bad = is_bad(b.m), empty = !bad && b.l == 0.f;
    const double log_l = log((double)b.l);
    sh.m = b.m;
    sh.log_l = log_l;
    if (a.stats != nullptr) {
      a.stats[(size_t)r * 2] = b.m;
      a.stats[(size_t)r * 2 + 1] = bad ? nan_f() : b.l;
    }
    a.entropy[r] = bad ? nan_f() : (empty ? 0.f : fmaxf((float)(log_l - kLn2 * (double)b.s / (double)b.l), 0.f));
    if (y >= 0) a.logprobs[r] = bad ? nan_f() : (empty ? -inf_f() : fminf((float)(kLn2 * rel2_exact(xy, b.m, c2) - log_l), 0.f));
  };
  if (cluster > 1) cluster_wait();   // every block of the cluster has started: its shared memory may be written
  // The last warp's: joins the block's sums.
  auto join = [&]() {
    Sums b = lane < warps ? sh.part[lane] : Sums{-FLT_MAX, 0.f, 0.f};
    b = warp_join(b, c2);
    if (cluster == 1) {
      tell(b);
    } else if (lane == 0) {
      store_to_cta(&sh.cta[rank][0], 0, b.m);
      store_to_cta(&sh.cta[rank][1], 0, b.l);
      store_to_cta(&sh.cta[rank][2], 0, b.s);
    }
  };
  if (!TOP && warp == warps - 1) join();
  if (TOP) {
    bool joined = false;
    // 2^j warps of which each has ceil(K / 2^j) threads: the 2^j-th largest over the warps, the best over j
    uint32_t lo, hi;
    {
      static_assert(kWarps == 8, "a lane for each warp and j");
      const int w = lane & 7, j = lane >> 3;
      const uint32_t mine = w < warps ? sh.least[j][w] : 0;
      int above = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t other = __shfl_sync(0xffffffffu, mine, (lane & 24) | i);
        above += other > mine || (other == mine && i < w);
      }
      lo = __reduce_max_sync(0xffffffffu, above == (1 << j) - 1 ? mine : 0);
      hi = __reduce_max_sync(0xffffffffu, w < warps ? sh.most[w] : 0);
    }
    int n = 0;
    if (!is_bad(key_value(hi)) && hi > kNegInfKey) {   // else this block has no alternatives
      lo = max(lo, kNegInfKey + 1);
      auto gather = [&]() {
        for (int s = 0; s < steps; ++s)
          if (groups[s * nt + tid] >= lo) {
            const int at = atomicAdd(&top.groups, 1);
            if (at < kGroups) top.group[at] = (s << 16) | tid;
          }
        __syncthreads();
      };
      gather();
      if (top.groups > min(kGroups, 2 * K + 32)) {
        lo = find_bound(top, groups, steps, lo, hi, K);     // (barriers between)
        if (tid == 0) top.groups = 0;
        __syncthreads();
        gather();
      }
      const float bound = key_value(lo);
      const int total = min(top.groups, kGroups) * kUnroll;
      // (the last warp has the row's sums to see to meanwhile)
      const int hands = warps > 1 ? nt - 32 : nt;
      if (warp == warps - 1) {
        join();
        joined = true;
      }
      for (int first = warp * 32; first < total && tid < hands; first += 2 * hands) {
        uint4 v[2];
        int vec[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int at = first + lane + u * hands, g = top.group[min(at, total - 1) / kUnroll];
          vec[u] = v0 + ((g >> 16) * kUnroll + at % kUnroll) * nt + (g & 0xffff);
          v[u] = at < total ? row.load(vec[u], v1) : Vec<T>::nothing();
        }
        constexpr int N = Vec<T>::N;
        uint32_t hits = 0;
#pragma unroll
        for (int i = 0; i < 2 * N; ++i)
          hits |= to_f(reinterpret_cast<const T*>(&v[i / N])[i % N]) >= bound ? 1u << i : 0u;
        int at = take_places(&top.n, __popc(hits));
        for (; __any_sync(0xffffffffu, hits != 0); hits &= hits - 1) {
          if (hits == 0) continue;
          const int i = __ffs(hits) - 1;
          const uint4 w = i < N ? v[0] : v[1];
          const float x = Vec<T>::one(w, i % N);
          if (at < kCandidates) top.list[at] = alt_key(order_key(x), row.col(i < N ? vec[0] : vec[1]) + i % N);
          ++at;
        }
      }
      __syncthreads();
      n = top.n;
      if (n > kCandidates || top.groups > kGroups) {
        __syncthreads();
        select_exactly<T>(top, row, v0, v1, K);
        n = top.n;
      }
    }
    if (warp == warps - 1 && !joined) join();
    rank_list(top, n, K, nt);
    if (cluster > 1)
      for (int k = tid; k < K; k += nt) store_to_cta(&lists[rank * K + k], 0, top.best[k]);
  }
  if (cluster > 1) {
    cluster_arrive();
    cluster_wait();
    if (rank != 0) return;
    // the last warp has the row's sums to see to, the others the lists
    const int hands = TOP && warps > 1 ? nt - 32 : nt;
    if (TOP && tid < hands) merge_lists(top, lists, cluster, K, hands);
    if (warp == warps - 1) {
      Sums b = lane < cluster ? Sums{sh.cta[lane][0], sh.cta[lane][1], sh.cta[lane][2]} : Sums{-FLT_MAX, 0.f, 0.f};
      tell(warp_join(b, c2));
    }
    if (TOP) __syncthreads();
  }
  if (!TOP) return;
  // (there was a barrier since tell())
  const bool bad = is_bad(sh.m);
  for (int k = tid; k < K; k += nt) {
    const uint64_t key = bad ? 0 : top.best[k];
    a.top_ids[(size_t)r * K + k] = key == 0 ? -1 : (int64_t)alt_col(key);
    const double lp = kLn2 * rel2_exact(key_value((uint32_t)(key >> 32)), sh.m, c2) - sh.log_l;
    a.top_logprobs[(size_t)r * K + k] = bad ? nan_f() : (key == 0 ? -inf_f() : fminf((float)lp, 0.f));
  }
}

// ------------------------------------------------------------------------------------------
// Backward: one block a segment of a row, all of it in flight at once. The columns named by the target and the alternatives
// get terms of their own: their logits are read before anything is written (the gradient may replace the logits), their
// results are written last. Segments that start at the row's first whole vector, with its ends apart, measured 175 us where
// this takes 169 (2048 x 128256 bf16, blocks of 256).
// ------------------------------------------------------------------------------------------
template <class T, bool ENTROPY>
__global__ void __launch_bounds__(kThreads, 4) logprobs_bwd_kernel(LogprobsArgs a, int segments) {
  constexpr int P = Vec<T>::kPairs;
  __shared__ int s_id[kHeadMaxTop + 4];
  __shared__ float s_c[kHeadMaxTop + 4], s_sum[kWarps];
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
  row.load_group(buf, v0, v0 + tid, nt, v1);
  // Entries: the alternatives, one a thread, and the first thread's second: the target.
  const int K = a.d_top != nullptr ? a.top_k : 0;
  int64_t id64[2] = {-1, -1};
  float c[2] = {0.f, 0.f};
  if (tid < K) {
    id64[0] = a.top_ids[(size_t)r * K + tid];
    c[0] = a.d_top[(size_t)r * K + tid];
  }
  if (tid == 0 && a.targets.p != nullptr && a.d_logprobs != nullptr) {
    id64[1] = load_id(a.targets, r);
    c[1] = a.d_logprobs[r];
  }
  int id[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const bool there = id64[i] >= 0 && id64[i] < a.V;
    id[i] = there ? (int)id64[i] : -1;
    c[i] = there ? c[i] : 0.f;
  }
  if (tid < K) {
    s_id[tid] = id[0];
    s_c[tid] = c[0];
  }
  if (tid < 4) {
    s_id[K + tid] = id[1];
    s_c[K + tid] = c[1];
  }
  const float sum = warp_sum(c[0] + c[1]);
  if ((tid & 31) == 0) s_sum[tid >> 5] = sum;
  __syncthreads();
  float g = 0.f;
  for (int w = 0; w < nt >> 5; ++w) g += s_sum[w];
  const float it = 1.f / a.temperature, c2 = scale2(a.temperature), inv_l = 1.f / l;
  // -p (g + h (ln p + H)) = 2^d (A + B d)
  const float h = ENTROPY ? a.d_entropy[r] : 0.f;
  const float B = ENTROPY ? -h * (float)kLn2 * inv_l * it : 0.f;
  const float A = -inv_l * it * (ENTROPY ? g + h * (float)((double)a.entropy[r] - log((double)l)) : g);
  T own[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (id[i] < row.col(v0) || id[i] >= row.col(v1)) id[i] = -1;
    own[i] = id[i] >= 0 ? row.x[id[i]] : T();
  }
  __syncthreads();
  const uint64_t B2 = pair(B, B), A2 = pair(A, A);
  const bool block_whole = v0 >= row.first_full && v0 + nt * kGradVecs <= min(v1, row.end_full) && out.vectors;
  auto dense = [&](auto rel) {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) {
      uint4 w;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        uint64_t d = rel(Vec<T>::get(buf[u], q));
        float d0, d1;
        unpair(d, d0, d1);
        if (ENTROPY) {
          d0 = fmaxf(d0, kLeast);
          d1 = fmaxf(d1, kLeast);
          d = pair(d0, d1);
        }
        const uint64_t e = pair(ex2(d0), ex2(d1));
        Vec<T>::put(w, q, mul2(e, ENTROPY ? fma2(B2, d, A2) : A2));
      }
      const int i = v0 + tid + u * nt;
      if (block_whole) *out.at(row, i) = w;
      else if (i < v1) out.store(row, i, w);
    }
  };
  if (is_far(m, c2)) dense(Rel2<true>(m, c2));
  else dense(Rel2<false>(m, c2));
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (id[i] < 0) continue;
    const float d = fmaxf(rel2(to_f(own[i]), m, c2), kLeast);
    float v = ex2(d) * fmaf(B, d, A);
    for (int k = 0; k <= K; k += 4) {     // (-1 behind the last)
#pragma unroll
      for (int u = 0; u < 4; ++u) v += s_id[k + u] == id[i] ? s_c[k + u] * it : 0.f;
    }
    from_f(v, out.p[id[i]]);
  }
}

// ------------------------------------------------------------------------------------------
// Launches
// ------------------------------------------------------------------------------------------
int threads_for(int vecs, int least) {
  const int n = ((vecs > least ? vecs : least) + 31) / 32 * 32;
  return n < kThreads ? n : kThreads;
}

template <class T>
void launch_fwd(const LogprobsArgs& a) {
  const int vecs = most_vecs<T>(a.logits, a.ld, a.rows, a.V);
  const bool top = a.top_k > 0;
  // Where every SM gets rows of its own, blocks of 128 threads (eight on an SM) even out better than 256 (four): without
  // alternatives 4096 x 128256 bf16 161 against 166 us, 999 x 50257 fp16 22.5 against 23.9, but 64 x 128256 fp32 13.2
  // against 10.2. The search for alternatives wants the threads where rows are long or few: 4096 x 128256, 64 of them,
  // 219 us with 256 threads, 255 with 128; 1024 x 32000 fp32, 20 of them, 35.7 and 31.7.
  const bool small = top ? (int64_t)a.rows * 128 * 2 > 1024 * (int64_t)a.sm_count && vecs <= 8192 : a.rows >= a.sm_count;
  const int threads = std::min(threads_for(vecs, 32), small ? 128 : kThreads);
  // Blocks a row: an SM takes 1024 threads; fewer rows than that are split as long as a block keeps a vector for each thread.
  int cluster = 1;
  while (cluster < kMaxCluster && (int64_t)a.rows * cluster * 2 * threads <= 1024 * (int64_t)a.sm_count && vecs / (cluster * 2) >= threads)
    cluster *= 2;
  while (cluster < kMaxCluster && vecs / cluster > 64 * threads * kUnroll) cluster *= 2;   // group maxima: 64 KB at most
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
  // Blocks of 128 threads, eight on an SM: 2048 x 128256 bf16 166.5 us, 999 x 50257 fp16 39.9; of 256: 169.1 and 42.4.
  const int threads = std::min(128, threads_for(vecs, a.d_top != nullptr ? a.top_k : 32));
  const int segments = (vecs + threads * kGradVecs - 1) / (threads * kGradVecs);
  if (a.d_entropy != nullptr) launch(logprobs_bwd_kernel<T, true>, a.rows, segments, false, threads, 0, a.stream, a, segments);
  else launch(logprobs_bwd_kernel<T, false>, a.rows, segments, false, threads, 0, a.stream, a, segments);
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

}  // namespace zx
