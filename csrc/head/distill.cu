// Distillation from a teacher of which K tokens' log-probabilities are known: for logits x [rows, V], z = x / temperature,
// p = softmax(z), teacher values v_k at the columns i_k:
//   renormalize: q = softmax(v);                    loss = sum q_k (log q_k - log p_{i_k})
//   bucket:      q = exp(v), q_r = max(0, 1 - sum q), p_r = the sum of p outside the columns;   + q_r (log q_r - log p_r)
//   temperature dloss/dx_j = s p_j - q_j  (bucket, outside the columns: p_j (s - q_r / p_r))
// where s is the sum of the weights in the loss: 1, but sum q where a bucket has nothing left (rounded values may add up to
// more than 1) or where the student has nothing outside, so that the bucket's part is not in the loss.
// Bound by the bytes of the logits, read once, and of the gradient. Measured on a B200 that copies 6557 GB/s, 64 of the
// teacher's tokens: loss and gradient of 4096 x 128256 bf16 400 us (5.2 TB/s), 4096 x 32000 fp32 170 (6.2), 4000 x 50257
// bf16 162 (4.9), 256 x 512 with 8 tokens 7.3 us; the loss alone of 4096 x 128256 235 us (4.5), its gradient from the
// statistics 319 (6.6). The alternatives named below were measured when the first of these took 391.
#include <algorithm>
#include <type_traits>
#include "rows.cuh"

namespace zx {

namespace {

constexpr int kEntries = kHeadMaxTop / 32;   // a lane's entries: k = lane + 32 i

// The teacher's entries of one row, held by a warp.
struct Entries {
  int id[kEntries];     // -1: absent
  float v[kEntries];    // the teacher's value
  float q[kEntries];    // weight
};
struct Teacher {
  bool live;            // the row counts
  double log_norm;      // log q_k = v_k - log_norm
  float q_rest;         // what the bucket has left
};

// As they lie in memory: nothing looks at them before take_entries, so that the loads are not waited for.
struct RawEntries {
  int64_t id[kEntries];
  uint32_t v[kEntries];
};
__device__ __forceinline__ void load_entries(const DistillArgs& a, int r, RawEntries& e) {
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    const int k = (threadIdx.x & 31) + 32 * i;
    const size_t at = (size_t)r * a.K + k;
    e.id[i] = -1;
    e.v[i] = 0;
    if (k < a.K) {
      if (a.ids.wide) e.id[i] = reinterpret_cast<const int64_t*>(a.ids.p)[at];
      else e.id[i] = reinterpret_cast<const int32_t*>(a.ids.p)[at];
      if (a.value_type == LOGIT_FP32) e.v[i] = reinterpret_cast<const uint32_t*>(a.values)[at];
      else e.v[i] = reinterpret_cast<const uint16_t*>(a.values)[at];
    }
  }
}
__device__ __forceinline__ void take_entries(const DistillArgs& a, const RawEntries& raw, Entries& e) {
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    const bool there = raw.id[i] >= 0 && raw.id[i] < a.V;
    float v = __uint_as_float(raw.v[i]);
    if (a.value_type == LOGIT_BF16) v = __uint_as_float(raw.v[i] << 16);
    if (a.value_type == LOGIT_FP16) v = __half2float(__ushort_as_half((unsigned short)raw.v[i]));
    e.id[i] = there ? (int)raw.id[i] : -1;
    e.v[i] = there ? v : -inf_f();
  }
}
// What a bucket has left, of which a peaked teacher leaves few digits in 32 bits. Called where that is less than a quarter (of
// more than that the roundings of a sum of 128 weights are below 2^-14): weights in 64 bits in every row made the loss alone
// of 4096 x 128256 bf16 253 us instead of 234.
__device__ __noinline__ float rest_in_64_bits(float4 v) {
  const double total = warp_sum((exp((double)v.x) + exp((double)v.y)) + (exp((double)v.z) + exp((double)v.w)));
  return total < 1. ? (float)(1. - total) : 0.f;
}
template <bool REST>
__device__ __forceinline__ Teacher weigh(const DistillArgs& a, Entries& e) {
  Teacher t;
  float vm = -inf_f();
  bool any = false;
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    vm = max_nan(vm, e.v[i]);
    any |= e.id[i] >= 0;
  }
  vm = warp_max_nan(vm);
  any = __any_sync(0xffffffffu, any);
  t.live = any && (a.bucket || vm != -inf_f());
  t.log_norm = 0.;
  t.q_rest = 0.f;
  const float base = a.bucket || !t.live ? 0.f : vm;
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    e.q[i] = e.id[i] >= 0 ? ex2((e.v[i] - base) * (float)kLog2e) : 0.f;
    total += e.q[i];
  }
  total = warp_sum(total);
  if (a.bucket) {
    t.q_rest = fmaxf(0.f, 1.f - total);
    static_assert(kEntries == 4, "by value");
    if (REST && t.q_rest < 0.25f) t.q_rest = rest_in_64_bits(make_float4(e.v[0], e.v[1], e.v[2], e.v[3]));    // (absent: -inf)
  } else if (t.live) {
    t.log_norm = (double)vm + log((double)total);
    const float norm = 1.f / total;
#pragma unroll
    for (int i = 0; i < kEntries; ++i) e.q[i] *= norm;
  }
  return t;
}
// The entries' weights with those of the same token added up, and whether an entry is the first with its token.
// Entries are few: each looks at all. s_id, s_w: [kHeadMaxTop] in shared memory for this warp.
__device__ __noinline__ void join_same(const Entries& e, int K, int* s_id, float* s_w, float (&q_all)[kEntries],
                                       bool (&first)[kEntries]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < kEntries; ++i) {
    s_id[lane + 32 * i] = e.id[i];
    s_w[lane + 32 * i] = e.q[i];
    q_all[i] = 0.f;
    first[i] = e.id[i] >= 0;
  }
  __syncwarp();
#pragma unroll 1
  for (int k = 0; k < K; ++k) {
    const int id = s_id[k];
    const float w = s_w[k];
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const bool same = id == e.id[i];
      q_all[i] += same ? w : 0.f;
      if (same && k < lane + 32 * i) first[i] = false;
    }
  }
  __syncwarp();
}

// Loss (and gradient): the blocks of a cluster share a row, each with a slice of it in shared memory from the first look
// to the gradient, so the logits are read once. The grid has a cluster for each row; one that is done with its row takes
// the row of a cluster that has not started (cluster launch control), so that the blocks' barriers and the entries of the
// next row are there when the slice is free. An auxiliary warp sees to that, starts the copy of the slice, takes the columns
// of the teacher's tokens out of it (-inf) when it is there, and weighs the next row's entries meanwhile. Four to six blocks
// on an SM, at different points of their rows, keep the memory busy: a block's own chain (copy, sums, exchange within the
// cluster, gradient) is several times the time in which the SM moves a slice. What bounds it: 9.4 instructions a logit and
// 2800 a block and row on the issue slots, and the shared memory that is filled. What it took the place of, 4096 x 128256:
// the slice in registers 864 us, two stages a block 924, one grid of clusters without taking over rows 578, a ring between
// warps that sum, write and copy 580, a row read again from the L2 cache by one block 441.
//
// The teacher's columns are kept apart so that the sum over all others is taken relative to their own maximum: the mass
// outside keeps its digits when the teacher's tokens have nearly all of it.
// stats = (maximum outside, coefficient of 2^d outside, maximum, s / l); the last is -1 for a row that is left out.
constexpr int kWorkers = 128;
constexpr int kWorkerWarps = kWorkers / 32;
constexpr int kCopy = 8192;    // bytes of one asynchronous copy

struct alignas(16) TeacherPart {   // of the teacher's tokens in a block's slice; moved in stores of 16 bytes
  float mt, lt, q, none;           // maximum, sum relative to it, sum of q_k
  double terms, weight;            // in the first block: sum of q_k (log q_k - ln 2 rel2(x_k)), sum of q_k
};
struct DistillShared {
  uint64_t full, ready, empty, exchanged[2], answered, told[2], taken[2];
  // of a row, from all blocks of the cluster: each worker warp's part, each auxiliary warp's part
  float2 outside[2][kMaxCluster * kWorkerWarps];
  TeacherPart teacher[2][kMaxCluster];
  uint4 answer;                // to the request for a row that has not started
  uint4 next[2];               // rows in turn: .x, or -1 after the last
  // from the auxiliary warp
  int row, live;               // row: -1 after the last
  float q_rest;
  int id[kHeadMaxTop];         // columns in this block's slice, or -1
  float x[kHeadMaxTop], q_all[kHeadMaxTop];
  int abort;
};

__device__ __forceinline__ void copy_in(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
// mbar_wait_cluster_w, which starts with a look at the clock, for what is mostly there already.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
#pragma unroll 1
  for (int i = 0; i < 256; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n\t"
        ".reg .pred P;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, P;\n\t"
        "}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    if (__all_sync(0xffffffffu, ok != 0)) return true;
  }
  return mbar_wait_cluster_w(bar, parity, abort_flag);
}
// 16 bytes into a block of the cluster, reported to its barrier when they are there (a store and a remote arrival would
// wait for the store's way back first).
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, float a, float b, float c, float d) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(to), "r"(bar),
               "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, double a, double b) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b64 [%0], {%2, %3}, [%1];" ::"r"(to), "r"(bar),
               "l"(__double_as_longlong(a)), "l"(__double_as_longlong(b))
               : "memory");
}
__device__ __forceinline__ void send(uint32_t to, uint32_t bar, float a, float b) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%2, %3}, [%1];" ::"r"(to), "r"(bar), "f"(a),
               "f"(b)
               : "memory");
}
// Asks for a cluster of this grid that has not started; the answer is 16 bytes of shared memory.
__device__ __forceinline__ void request_cluster(uint4* answer, uint64_t* bar) {
  mbar_expect_tx(bar, 16);
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(smem_u32(answer)),
               "r"(smem_u32(bar))
               : "memory");
}
// Its first block, or -1: there is none, and no other request may follow.
__device__ __forceinline__ int answered_block(const uint4* answer) {
  uint32_t got, block;
  asm volatile(
      "{\n\t"
      ".reg .pred p;\n\t"
      ".reg .b128 h;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, _, _, _}, h;\n\t"
      "}\n"
      : "=r"(got), "=r"(block)
      : "r"(smem_u32(answer))
      : "memory");
  fence_proxy_async_smem();            // read before the next one may be written
  return got ? (int)block : -1;
}
constexpr int kSiteCopy = 51, kSiteReady = 52, kSiteEmpty = 53, kSiteExchange = 54, kSiteRow = 55;

template <class T>
__device__ __forceinline__ void distill_auxiliary(const DistillArgs& a, DistillShared& sh, uint4* stage, int cluster, int rank,
                                                  float c2) {
  constexpr int N = Vec<T>::N;
  using Raw = typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type;
  const int lane = threadIdx.x & 31;
  T* elems = reinterpret_cast<T*>(stage);
  volatile Raw* raw = reinterpret_cast<volatile Raw*>(stage);
  Entries e;
  int r = blockIdx.x / cluster;
  int copies = 0, requests = 0, answers = 0;     // begun and (the answers) seen
  int live_rows = 0;
  // A wait ran out: nothing of this block's stays in flight (bounded as well).
  auto leave = [&](int site) {
    if (lane == 0) report(a.status, ZX_ERR_TIMEOUT, site, r);
    int none = 0;
    if (copies > 0) mbar_wait(&sh.full, (copies - 1) & 1, &none);
    if (requests > answers) mbar_wait(&sh.answered, answers & 1, &none);
    __syncwarp();
  };
  if (rank == 0) {
    if (lane == 0) request_cluster(&sh.answer, &sh.answered);
    ++requests;
  }
  RawEntries next;
  load_entries(a, r, next);
  take_entries(a, next, e);
  Teacher t = weigh<true>(a, e);
  // The first block of the cluster passes the answer to request i on to all blocks (row i + 1 of this cluster).
  auto pass_on = [&](int i) {
    if (!mbar_wait_w(&sh.answered, i & 1, &sh.abort)) return false;
    ++answers;
    const int block = answered_block(&sh.answer), row = block < 0 ? -1 : block / cluster;
    if (cluster > 1) {
      if (i >= 2 && !wait_cluster(&sh.taken[i & 1], (i >> 1) & 1 ^ 1, &sh.abort)) return false;
      if (lane < cluster)
        send(map_to_cta(&sh.next[i & 1], lane), map_to_cta(&sh.told[i & 1], lane), __int_as_float(row), 0.f, 0.f, 0.f);
    } else if (lane == 0) {
      sh.next[i & 1].x = (uint32_t)row;
    }
    __syncwarp();
    return true;
  };
  if (rank == 0 && !pass_on(0)) return leave(kSiteRow);
  for (int n = 0;; ++n) {
    const Row<T> row(a.logits, r, a.ld, a.V);
    const int per = (row.vecs + cluster - 1) / cluster;
    const int v0 = min(rank * per, row.vecs), v1 = min(v0 + per, row.vecs);
    const int w0 = max(v0, row.first_full), w1 = min(v1, row.end_full);
    if (n >= 1) {
      // the workers still have the slice: into the L2 cache with the next one meanwhile
      if (lane == 0 && t.live && w1 > w0) prefetch_l2(row.at(w0), (uint32_t)(w1 - w0) * 16);
      if (!mbar_wait_w(&sh.empty, (n - 1) & 1, &sh.abort)) return leave(kSiteEmpty);
    }
    if (lane == 0) {
      if (t.live && w1 > w0) {
        fence_proxy_async_smem();     // the stage was written by threads before
        mbar_expect_tx(&sh.full, (uint32_t)(w1 - w0) * 16);
        for (int v = w0; v < w1; v += kCopy / 16)
          copy_in(stage + (v - v0), row.at(v), (uint32_t)min(kCopy, (w1 - v) * 16), &sh.full);
      } else {
        mbar_arrive(&sh.full);
      }
    }
    ++copies;
    __syncwarp();
    // the next row
    if (cluster > 1) {
      if (lane == 0) mbar_expect_tx(&sh.told[n & 1], 16);
      __syncwarp();
      if (!wait_cluster(&sh.told[n & 1], (n >> 1) & 1, &sh.abort)) return leave(kSiteRow);
    }
    const int next_r = (int)sh.next[n & 1].x;
    __syncwarp();
    if (rank == 0 && next_r >= 0) {
      if (lane == 0) request_cluster(&sh.answer, &sh.answered);
      ++requests;
    }
    if (next_r >= 0) load_entries(a, next_r, next);
    // partial vectors at the ends of the row
    if (t.live) {
      if (lane == 0 && v0 == 0 && row.first_full > 0) stage[0] = row.edge(0);
      if (lane == 1 && v1 == row.vecs && v1 > v0 && !row.whole(v1 - 1) && v1 - 1 >= row.first_full)
        stage[v1 - 1 - v0] = row.edge(v1 - 1);
    }
    if (!mbar_wait_w(&sh.full, n & 1, &sh.abort)) return leave(kSiteCopy);
    __syncwarp();
    if (t.live) {
      int at[kEntries];
      float x[kEntries], q_all[kEntries];
      bool first[kEntries];
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        const int v = e.id[i] >= 0 ? row.vec_of(e.id[i]) : -1;
        at[i] = v >= v0 && v < v1 ? e.id[i] + row.lead - v0 * N : -1;
        x[i] = at[i] >= 0 ? to_f(elems[at[i]]) : -inf_f();
        q_all[i] = e.q[i];
        first[i] = at[i] >= 0;
      }
      __syncwarp();
      // a token that is named twice: each entry leaves its number in the column, one of them finds another's
#pragma unroll
      for (int i = 0; i < kEntries; ++i)
        if (at[i] >= 0) raw[at[i]] = (Raw)(lane + 32 * i);
      __syncwarp();
      bool twice = false;
#pragma unroll
      for (int i = 0; i < kEntries; ++i)
        if (at[i] >= 0) twice |= raw[at[i]] != (Raw)(lane + 32 * i);
      if (__any_sync(0xffffffffu, twice)) {
        join_same(e, a.K, sh.id, sh.x, q_all, first);
#pragma unroll
        for (int i = 0; i < kEntries; ++i) first[i] = first[i] && at[i] >= 0;
      }
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        if (at[i] >= 0) from_f(-inf_f(), elems[at[i]]);
        sh.id[lane + 32 * i] = first[i] ? e.id[i] : -1;
        sh.x[lane + 32 * i] = x[i];
        sh.q_all[lane + 32 * i] = q_all[i];
      }
      if (lane == 0) {
        sh.row = r;
        sh.live = 1;
        sh.q_rest = t.q_rest;
      }
      mbar_arrive_warp(&sh.ready);
      const int xc = live_rows & 1;
      // what all blocks send to this one: 8 bytes a worker warp, 16 an auxiliary warp, to the first block 16 more for the loss
      if (cluster > 1 && lane == 0) mbar_expect_tx(&sh.exchanged[xc], cluster * (8 * kWorkerWarps + (rank == 0 ? 32 : 16)));
      ++live_rows;
      float mt = -FLT_MAX;
#pragma unroll
      for (int i = 0; i < kEntries; ++i) mt = max_nan(mt, x[i]);
      mt = warp_max_nan(mt);
      float lt = 0.f;
      double terms = 0., weight = 0.;
#pragma unroll
      for (int i = 0; i < kEntries; ++i) {
        if (first[i]) lt += ex2(rel2(x[i], mt, c2));
        if (at[i] >= 0 && e.q[i] != 0.f) {
          const double z = x[i] == -inf_f() ? -(double)inf_f() : kLn2 * rel2_exact(x[i], mt, c2);
          weight += (double)e.q[i];
          terms += (double)e.q[i] * ((double)e.v[i] - t.log_norm - z);
        }
      }
      lt = warp_sum(lt);
      terms = warp_sum(terms);
      weight = warp_sum(weight);
      if (cluster > 1) {
        if (lane < cluster) {
          const uint32_t to = map_to_cta(&sh.teacher[xc][rank], lane), bar = map_to_cta(&sh.exchanged[xc], lane);
          send(to, bar, mt, lt, (float)weight, 0.f);
          if (lane == 0) send(to + 16, bar, terms, weight);
        }
        __syncwarp();
      } else {
        // launched without a cluster: such a store is not allowed there, not even to the block itself
        if (lane == 0) sh.teacher[xc][0] = TeacherPart{mt, lt, (float)weight, 0.f, terms, weight};
        mbar_arrive_warp(&sh.exchanged[xc]);
      }
    } else {
      if (lane == 0) {
        sh.row = r;
        sh.live = 0;
      }
      mbar_arrive_warp(&sh.ready);
    }
    if (next_r < 0) {
      if (!mbar_wait_w(&sh.empty, n & 1, &sh.abort)) return leave(kSiteEmpty);
      if (lane == 0) sh.row = -1;
      mbar_arrive_warp(&sh.ready);
      return;
    }
    r = next_r;
    take_entries(a, next, e);
    t = weigh<true>(a, e);
    // The first block may write sh.next[n & 1] again: a release, since nothing else orders the read before that where rows
    // are left out. It waits for copies in flight: where the word is read, or behind the start of the next copy, 1024 x 32000
    // fp32 with 128 entries takes 63 to 67 us, here, while the workers have the slice, 55 to 57.
    if (cluster > 1) mbar_arrive_warp_cluster(map_to_cta(&sh.taken[n & 1], 0));
    if (rank == 0 && !pass_on(n + 1)) return leave(kSiteRow);
  }
}

// Vectors of the slice into the running maximum and sum.
template <class T, int U, class Rel>
__device__ __forceinline__ void sum_outside(const uint4 (&v)[U], Rel rel, float gap, uint64_t (&l2)[2]) {
  const float f = ex2(gap);
  l2[0] = mul2(l2[0], pair(f, f));
  l2[1] = mul2(l2[1], pair(f, f));
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int q = 0; q < Vec<T>::kPairs; ++q) {
      float d0, d1;
      unpair(rel(Vec<T>::get(v[u], q)), d0, d1);
      l2[q & 1] = add2(l2[q & 1], pair(ex2(d0), ex2(d1)));
    }
}
// The same, for rows that are far from zero (apart, so that it costs the others nothing).
template <class T>
__device__ __noinline__ uint64_t far_outside(const uint4* p, int U, float m, float M, uint64_t l, float c2) {
  uint64_t l2[2] = {l, 0};
  for (int u = 0; u < U; ++u) {
    const uint4 v[1] = {p[u * kWorkers]};
    const float gap = u == 0 ? gap2_far(m, M, c2) : 0.f;
    if (is_far(M, c2)) sum_outside<T, 1>(v, Rel2<true>(M, c2), gap, l2);
    else sum_outside<T, 1>(v, Rel2<false>(M, c2), gap, l2);
  }
  return add2(l2[0], l2[1]);
}
template <class T, int U>
__device__ __forceinline__ void add_outside(const uint4* p, float& m, uint64_t (&l2)[2], float c2) {
  uint4 v[U];
#pragma unroll
  for (int u = 0; u < U; ++u) v[u] = p[u * kWorkers];
  uint32_t mw = Vec<T>::max_w(v[0]);
#pragma unroll
  for (int u = 1; u < U; ++u) mw = Elem<T>::max_w(mw, Vec<T>::max_w(v[u]));
  const float M = max_nan(m, Vec<T>::max_of(mw)), R = ref2(M, c2);
  if (plain_gap(R)) {
    sum_outside<T, U>(v, Rel2<false>(M, c2), gap2_plain(m, R, c2), l2);
  } else {
    l2[0] = far_outside<T>(p, U, m, M, add2(l2[0], l2[1]), c2);
    l2[1] = 0;
  }
  m = M;
}

template <class T, bool WRITE>
__global__ void __launch_bounds__(kWorkers + 32, 6) distill_kernel(DistillArgs a, int cluster) {
  constexpr int P = Vec<T>::kPairs;
  extern __shared__ __align__(16) unsigned char dynamic[];    // the slice
  __shared__ DistillShared sh;
  uint4* stage = reinterpret_cast<uint4*>(dynamic);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rank = blockIdx.x % cluster;
  if (tid == 0) {
    mbar_init(&sh.full, 1);
    mbar_init(&sh.ready, 1);
    mbar_init(&sh.empty, kWorkerWarps);
    mbar_init(&sh.answered, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.exchanged[i], cluster > 1 ? 1 : 1 + kWorkerWarps);
      mbar_init(&sh.told[i], 1);
      mbar_init(&sh.taken[i], cluster);
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  __syncthreads();
  if (cluster > 1) cluster_sync();      // barriers of all blocks are there
  const float c2 = scale2(a.temperature);

  if (warp == kWorkerWarps) {
    distill_auxiliary<T>(a, sh, stage, cluster, rank, c2);
  } else {
    // The worker warps go their own ways: what they need of one another they get through the exchange.
    for (int n = 0, live_rows = 0;; ++n) {
      bool ok = mbar_wait_w(&sh.ready, n & 1, &sh.abort);
      const int r = sh.row;
      if (ok && r < 0) break;
      ok = ok && mbar_wait_w(&sh.full, n & 1, &sh.abort);
      if (!ok) {
        if (lane == 0) report(a.status, ZX_ERR_TIMEOUT, kSiteReady, r);
        break;
      }
      const Row<T> row(a.logits, r, a.ld, a.V);
      const int per = (row.vecs + cluster - 1) / cluster;
      const int v0 = min(rank * per, row.vecs), len = min(v0 + per, row.vecs) - v0;
      const OutRow<T> out(WRITE ? a.d_logits : const_cast<void*>(a.logits), r, WRITE ? a.d_ld : a.ld, row);
      if (!sh.live) {
        if (rank == 0 && tid == 0) {
          a.loss[r] = 0.f;
          if (!WRITE) reinterpret_cast<float4*>(a.stats)[r] = make_float4(0.f, 0.f, 0.f, -1.f);
        }
        mbar_arrive_warp(&sh.empty);
        if (WRITE)
          for (int i = tid; i < len; i += kWorkers) out.store(row, v0 + i, make_uint4(0, 0, 0, 0));
        continue;
      }
      // maximum and sum of what is outside
      float mr = -FLT_MAX, lr = 0.f;
      {
        uint64_t l2[2] = {0, 0};
        int i = tid;
#pragma unroll 1
        for (; i + 3 * kWorkers < len; i += 4 * kWorkers) add_outside<T, 4>(stage + i, mr, l2, c2);
#pragma unroll 1
        for (; i < len; i += kWorkers) add_outside<T, 1>(stage + i, mr, l2, c2);
        float x0, x1;
        unpair(add2(l2[0], l2[1]), x0, x1);
        const float M = warp_max_nan(mr);
        lr = warp_sum((x0 + x1) * ex2(gap2(mr, M, c2)));
        mr = M;
      }
      const int xc = live_rows & 1;
      if (cluster > 1) {
        if (lane < cluster)
          send(map_to_cta(&sh.outside[xc][rank * kWorkerWarps + warp], lane), map_to_cta(&sh.exchanged[xc], lane), mr, lr);
        __syncwarp();
      } else {
        if (lane == 0) sh.outside[xc][warp] = make_float2(mr, lr);
        mbar_arrive_warp(&sh.exchanged[xc]);
      }
      // what the last steps need of the auxiliary warp's words, which are free with the slice
      int id[kEntries];
      float x[kEntries], q_all[kEntries];
      if (WRITE) {
#pragma unroll
        for (int i = 0; i < kEntries; ++i) {
          id[i] = sh.id[lane + 32 * i];
          x[i] = sh.x[lane + 32 * i];
          q_all[i] = sh.q_all[lane + 32 * i];
        }
      }
      const float q_rest = sh.q_rest;
      if (!wait_cluster(&sh.exchanged[xc], (live_rows >> 1) & 1, &sh.abort)) {
        if (lane == 0) report(a.status, ZX_ERR_TIMEOUT, kSiteExchange, r);
        break;
      }
      ++live_rows;
      static_assert(kMaxCluster * kWorkerWarps == 32 && kMaxCluster == 8, "a part a lane");
      const float2 part = lane < cluster * kWorkerWarps ? sh.outside[xc][lane] : make_float2(-FLT_MAX, 0.f);
      const TeacherPart& tp = sh.teacher[xc][(lane & 7) < cluster ? lane & 7 : 0];
      const float tm = (lane & 7) < cluster ? tp.mt : -FLT_MAX;
      mr = warp_max_nan(part.x);
      const float m = max_nan(mr, warp_max_nan<8>(tm)), Rr = ref2(mr, c2), R = ref2(m, c2);
      float lt, share;
      auto join = [&](float to_mr, float t_to_m, float r_to_m) {
        lr = warp_sum(part.y * ex2(to_mr));
        lt = warp_sum<8>((lane & 7) < cluster ? tp.lt * ex2(t_to_m) : 0.f);
        share = ex2(r_to_m);
      };
      if (plain_gap(Rr) && plain_gap(R)) join(gap2_plain(part.x, Rr, c2), gap2_plain(tm, R, c2), gap2_plain(mr, R, c2));
      else join(gap2_far(part.x, mr, c2), gap2_far(tm, m, c2), gap2_far(mr, m, c2));
      const float l = lt + lr * share;
      const bool bad = is_bad(m);
      float weights = 1.f;      // s
      if (a.bucket && !(q_rest > 0.f && lr != 0.f)) {
        weights = 0.f;
        for (int c = 0; c < cluster; ++c) weights += sh.teacher[xc][c].q;
      }
      const float inv_l = bad ? nan_f() : (l == 0.f ? 0.f : weights / l);
      const float coef = bad ? nan_f() : (lr == 0.f ? 0.f : share * inv_l - q_rest / lr);
      if (WRITE) {
        const float w = a.grad_scale / a.temperature;
        const uint64_t w2 = pair(w * coef, w * coef);
        // whole vectors go out as such where the output's rows have the logits' alignment; the others one by one
        const int i_end = out.vectors ? min(v0 + len, row.end_full) - v0 : 0;
        const int i_first = out.vectors ? max(row.first_full - v0, 0) : 0;
        auto dense = [&](auto rel) {
          auto one = [&](int i) {
            const uint4 v = stage[i];
            uint4 g;
#pragma unroll
            for (int q = 0; q < P; ++q) {
              float d0, d1;
              unpair(rel(Vec<T>::get(v, q)), d0, d1);
              Vec<T>::put(g, q, mul2(pair(ex2(d0), ex2(d1)), w2));
            }
            return g;
          };
          int i = tid;
          if (i < i_first || i_end == 0) {
            for (; i < len && (i < i_first || i_end == 0); i += kWorkers) out.store(row, v0 + i, one(i));
          }
          uint4* p = out.at(row, v0 + i);
#pragma unroll 1
          for (; i + 3 * kWorkers < i_end; i += 4 * kWorkers, p += 4 * kWorkers) {
            uint4 g[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) g[u] = one(i + u * kWorkers);
#pragma unroll
            for (int u = 0; u < 4; ++u) p[u * kWorkers] = g[u];
          }
#pragma unroll 1
          for (; i < i_end; i += kWorkers, p += kWorkers) *p = one(i);
          for (; i < len; i += kWorkers) out.store(row, v0 + i, one(i));
        };
        if (is_far(mr, c2)) dense(Rel2<true>(mr, c2));
        else dense(Rel2<false>(mr, c2));
        mbar_arrive_warp(&sh.empty);
        // the teacher's columns among this warp's vectors, written as 0 so far
#pragma unroll
        for (int i = 0; i < kEntries; ++i) {
          if (id[i] < 0 || ((row.vec_of(id[i]) - v0) % kWorkers) / 32 != warp) continue;
          const float p = inv_l * ex2(rel2(x[i], m, c2));
          from_f(w * (p - q_all[i]), out.p[id[i]]);
        }
        __syncwarp();
      } else {
        mbar_arrive_warp(&sh.empty);
      }
      if (rank == 0 && tid == kWorkers - 32) {
        const double log_l = log((double)l);
        double loss = 0.;
        // - log p_k = log l - (x_k - m) / t; a student with nothing has infinite terms already
        for (int c = 0; c < cluster; ++c) {
          const TeacherPart& p = sh.teacher[xc][c];
          loss += p.terms;
          if (l != 0.f && p.weight != 0.) loss += p.weight * (log_l - kLn2 * gap2_exact(p.mt, m, c2));
        }
        if (q_rest > 0.f && lr != 0.f) {
          const double lp = kLn2 * gap2_exact(mr, m, c2) + log((double)lr) - log_l;
          loss += (double)q_rest * (log((double)q_rest) - lp);
        }
        a.loss[r] = bad ? nan_f() : (float)loss;
        if (!WRITE) reinterpret_cast<float4*>(a.stats)[r] = make_float4(mr, coef, m, inv_l);
      }
      __syncwarp();
    }
  }
  // no block leaves while another may still write to it
  __syncthreads();
  if (cluster > 1) cluster_sync();
}

// ------------------------------------------------------------------------------------------
// Gradient from the forward's statistics, one block a segment of a row. The first warps hold the teacher's entries.
// ------------------------------------------------------------------------------------------
// Blocks of 128 threads: 365 us instead of 317 for 4096 x 128256 bf16 (the entries are a warp's work in each block).
constexpr int kThreads = 256;
constexpr int kGradVecs = 8;    // vectors of a thread, all in flight

template <class T>
__global__ void __launch_bounds__(kThreads, 4) distill_bwd_kernel(DistillArgs a, int segments) {
  constexpr int P = Vec<T>::kPairs, N = Vec<T>::N;
  __shared__ uint32_t marks[kThreads * kGradVecs * N / 32];   // a bit for each column of the segment: named by the teacher
  __shared__ int s_id[kHeadMaxTop];
  __shared__ float s_w[kHeadMaxTop];
  const int tid = threadIdx.x, lane = tid & 31;
  const int r = blockIdx.x / segments;
  const Row<T> row(a.logits, r, a.ld, a.V);
  const OutRow<T> out(a.d_logits, r, a.d_ld, row);
  const int v0 = (blockIdx.x % segments) * kThreads * kGradVecs, v1 = min(v0 + kThreads * kGradVecs, row.vecs);
  const float4 st = reinterpret_cast<const float4*>(a.stats)[r];
  if (st.w < 0.f) {
    for (int i = v0 + tid; i < v1; i += kThreads) out.store(row, i, make_uint4(0, 0, 0, 0));
    return;
  }
  RawEntries raw;
  if (tid < 32) load_entries(a, r, raw);
  uint4 buf[kGradVecs];
  row.load_group(buf, v0, v0 + tid, kThreads, v1);
  for (int i = tid; i < kThreads * kGradVecs * N / 32; i += kThreads) marks[i] = 0;
  __syncthreads();
  const float mr = st.x, coef = st.y, m = st.z, inv_l = st.w;
  const float c2 = scale2(a.temperature), w = a.d_loss[r] / a.temperature;
  if (tid < 32) {
    Entries e;
    float q_all[kEntries];
    bool first[kEntries];
    take_entries(a, raw, e);
    weigh<false>(a, e);      // (the statistics have what the bucket has left)
    bool again = false;
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      const int v = e.id[i] >= 0 ? row.vec_of(e.id[i]) : -1;
      first[i] = v >= v0 && v < v1;
      q_all[i] = e.q[i];
      if (first[i]) {
        const int at = e.id[i] + row.lead - v0 * N;
        again |= (atomicOr(&marks[at >> 5], 1u << (at & 31)) >> (at & 31)) & 1u;
      }
    }
    if (__any_sync(0xffffffffu, again)) {
      bool here[kEntries];
#pragma unroll
      for (int i = 0; i < kEntries; ++i) here[i] = first[i];
      join_same(e, a.K, s_id, s_w, q_all, first);
#pragma unroll
      for (int i = 0; i < kEntries; ++i) first[i] = first[i] && here[i];
    }
#pragma unroll
    for (int i = 0; i < kEntries; ++i) {
      s_id[lane + 32 * i] = first[i] ? e.id[i] : -1;
      if (first[i]) s_w[lane + 32 * i] = w * (inv_l * ex2(rel2(to_f(row.x[e.id[i]]), m, c2)) - q_all[i]);
    }
  }
  __syncthreads();   // those logits have been read: they may be overwritten
  const uint64_t w2 = pair(w * coef, w * coef);
  const bool block_whole = v0 >= row.first_full && v0 + kThreads * kGradVecs <= min(v1, row.end_full) && out.vectors;
  auto dense = [&](auto rel) {
#pragma unroll
    for (int u = 0; u < kGradVecs; ++u) {
      uint4 g;
#pragma unroll
      for (int q = 0; q < P; ++q) {
        float d0, d1;
        unpair(rel(Vec<T>::get(buf[u], q)), d0, d1);
        // (anything for the teacher's tokens, which may lie above the maximum of the others: they are written below)
        Vec<T>::put(g, q, mul2(pair(ex2(d0), ex2(d1)), w2));
      }
      const int i = v0 + tid + u * kThreads;
      if (block_whole) *out.at(row, i) = g;
      else if (i < v1) out.store(row, i, g);
    }
  };
  if (is_far(mr, c2)) dense(Rel2<true>(mr, c2));
  else dense(Rel2<false>(mr, c2));
  __syncthreads();
  if (tid < kHeadMaxTop && s_id[tid] >= 0) from_f(s_w[tid], out.p[s_id[tid]]);
}

// ------------------------------------------------------------------------------------------
// Launches
// ------------------------------------------------------------------------------------------
// Blocks a row. What counts is how many bytes of slices an SM holds, and then how few blocks they are in (each has its
// fixed work): the largest sum over four to six blocks, fewer blocks unless more hold a sixteenth more.
// 4096 x 128256 bf16: six blocks a row (five slices of 43 KB on an SM) 392 us, five 403, four and eight (192 KB held) 437
// and 433; 4000 x 50257: two (four of 50 KB) 163, three (six of 34 KB) 181, one (two of 100 KB) 192, four (six of 25 KB) 196;
// 4096 x 32000 fp32: three 170, two and four 173. Five and seven are left out: seven measured 262 us where six took 243
// (2048 x 151936), five never was the best.
// Few rows are split further, as long as the grid stays below five blocks an SM and a worker has a vector: 150 x 50257 takes
// 15.3 us with four blocks a row, 16.3 with two, 19.1 with eight.
int blocks_a_row(int vecs, int rows, int sm_count) {
  constexpr int kSizes[] = {1, 2, 3, 4, 6, 8};
  constexpr int kSmemOfSm = 228 * 1024, kOverhead = 1024 + (int)sizeof(DistillShared);
  int best = kMaxCluster, held = 0;
  for (int c : kSizes) {
    const int slice = (vecs + c - 1) / c * 16, n = std::min(6, kSmemOfSm / (slice + kOverhead));
    if (n >= 4 && n * slice > held + held / 16) {
      best = c;
      held = n * slice;
    }
  }
  for (int c : kSizes)
    if (c > best && (int64_t)rows * c <= 5 * sm_count && vecs / c >= kWorkers) best = c;
  return best;
}
template <class T, bool WRITE>
void launch_distill(const DistillArgs& a) {
  const int vecs = most_vecs<T>(a.logits, a.ld, a.rows, a.V);
  const int cluster = blocks_a_row(vecs, a.rows, a.sm_count);
  const int smem = (vecs + cluster - 1) / cluster * 16;
  launch(distill_kernel<T, WRITE>, a.rows, cluster, true, kWorkers + 32, smem, a.stream, a, cluster);
}

}  // namespace

void launch_distill_fwd(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { launch_distill<decltype(t), false>(a); });
}
void launch_distill_bwd(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) {
    using T = decltype(t);
    const int segments = (most_vecs<T>(a.logits, a.ld, a.rows, a.V) + kThreads * kGradVecs - 1) / (kThreads * kGradVecs);
    launch(distill_bwd_kernel<T>, a.rows, segments, false, kThreads, 0, a.stream, a, segments);
  });
}
void launch_distill_fwd_bwd(const DistillArgs& a) {
  if (a.rows == 0) return;
  by_type(a.type, [&](auto t) { launch_distill<decltype(t), true>(a); });
}

}  // namespace zx
