// Verification of drafted tokens by rejection sampling, from given random numbers.
//
// For each sequence: draft i (token x) is kept while u_i * q_i(x) < p_i(x), p the target's probabilities and q the draft
// model's (1 at x for drafts without probabilities); the products are exact in 64 bits.  At the first draft turned down
// one more token is drawn from max(p - q, 0), and from p when every draft was kept, or when p <= q everywhere: the first v with
// sum_{w <= v} weight(w) > u * sum(weight).  Sums are 64-bit: a token is decided by where u falls between neighbouring
// sums of up to 10^5 terms, which 32 bits place wrongly about once in a hundred draws.  No atomics: every sum has a fixed order.
//
// Bound by HBM: one row of p and one of q per sequence (the other rows are touched at one entry each).  ONE CLUSTER PER
// SEQUENCE, in one launch and without a workspace: each block sums a slice of the row, one contiguous segment per warp,
// the segment sums are exchanged through distributed shared memory, and the block whose segment holds the drawn point
// reads that segment again (from L2), a sixteenth for each warp, to find the token.  What stays beside the reading is the
// chain ids -> p(x), q(x) -> rows -> exchange -> search, each step a trip to memory or across the cluster: one sequence
// takes 5.3 us with 2000 entries, 7.1 with 32000, 10 with 163840, 64 of those 26 (one launch behind another).
//
// Four blocks of 512 threads on an SM, two loads of each row ahead: 64 sequences of 163840 entries with q (84 MB) take
// 31 us from launch to end, 18 of them the chain and the launch.  Two blocks of 64 registers with four loads ahead take
// 35 us (200 sequences: 94 against 70), three of 40 registers 35, and one warp for the search 5 us more.
#include <cooperative_groups.h>

#include "k3g_device.cuh"
#include "k3g_host.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kThreads = 512, kSegs = kThreads / 32, kMaxCluster = 8, kMaxSteps = 32;
constexpr int kBatch = 2;

struct Rows {                       // the row that is sampled from: weight(v) = p[v], or max(p[v] - q(v), 0)
  const float* p;
  const float* q;                   // null: q is 1 at `hot` and 0 elsewhere (hot < 0: 0 everywhere, the weight is p)
  int hot;
};
__device__ __forceinline__ double weight(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 && d < (double)INFINITY ? d : 0.0;          // NaN and infinite entries weigh nothing
}
__device__ __forceinline__ float q_at(const Rows& r, int v) { return r.q ? k3g::ld_ordered(r.q + v) : (v == r.hot ? 1.f : 0.f); }

// Weights of elements v .. v + 3 (those below `end`).
template <bool VEC>
__device__ __forceinline__ void weights4(const Rows& r, int v, int end, double (&w)[4]) {
  float p[4] = {0.f, 0.f, 0.f, 0.f}, q[4] = {0.f, 0.f, 0.f, 0.f};
  if (VEC && v + 4 <= end) {
    const float4 a = k3g::ld_ordered(reinterpret_cast<const float4*>(r.p + v));
    p[0] = a.x; p[1] = a.y; p[2] = a.z; p[3] = a.w;
    if (r.q) {
      const float4 b = k3g::ld_ordered(reinterpret_cast<const float4*>(r.q + v));
      q[0] = b.x; q[1] = b.y; q[2] = b.z; q[3] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = v + j == r.hot ? 1.f : 0.f;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (v + j < end) { p[j] = k3g::ld_ordered(r.p + v + j); q[j] = q_at(r, v + j); }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = weight(p[j], q[j]);
}

__device__ __forceinline__ double warp_sum(double x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

__device__ __forceinline__ double lane_scan(double x, int lane) {   // sum of the lanes up to and including this one
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// Lane l has the sums of parts 4 l .. 4 l + 3, and with `upto` their running sum (`start` before the first).  The part in
// which it passes `point`, else the last that weighs anything, -1 if none does; `base`: the running sum before it.
__device__ __forceinline__ int part_of(const double (&part)[4], double upto, double point, int lane, double& base, double start = 0.0) {
  double at = __shfl_up_sync(0xffffffffu, upto, 1);
  if (lane == 0) at = start;
  int hit = -1, top = -1;
  double hit_base = 0.0, top_base = 0.0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (part[j] > 0.0) {
      top = 4 * lane + j; top_base = at;
      if (hit < 0 && at + part[j] > point) { hit = top; hit_base = at; }
    }
    at += part[j];
  }
  const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), tops = __ballot_sync(0xffffffffu, top >= 0);
  const int from = hits ? __ffs(hits) - 1 : tops ? 31 - __clz(tops) : 0;
  base = __shfl_sync(0xffffffffu, hits ? hit_base : top_base, from);
  return __shfl_sync(0xffffffffu, hits ? hit : top, from);
}

// A function of its own: inlined at both places the kernel needs more than the 32 registers with which four blocks fit an SM.
template <bool VEC>
__device__ __noinline__ double segment_sum(const Rows r, int lo, int hi, int lane) {
  double s = 0.0;
  int v = lo + 4 * lane;
  if (VEC && r.q) {                                          // kBatch loads of each row are on their way before the first is used
    for (; v + 128 * (kBatch - 1) + 4 <= hi; v += 128 * kBatch) {
      float4 p[kBatch], q[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        p[j] = k3g::ld_ordered(reinterpret_cast<const float4*>(r.p + v + 128 * j));
        q[j] = k3g::ld_ordered(reinterpret_cast<const float4*>(r.q + v + 128 * j));
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) s += (weight(p[j].x, q[j].x) + weight(p[j].y, q[j].y)) + (weight(p[j].z, q[j].z) + weight(p[j].w, q[j].w));
    }
  }
#pragma unroll 4
  for (; v < hi; v += 128) {
    double w[4];
    weights4<VEC>(r, v, hi, w);
    s += (w[0] + w[1]) + (w[2] + w[3]);
  }
  return warp_sum(s);
}

// First element of [lo, hi) whose running sum, on top of `base`, passes `point`; the last one with a weight if rounding
// keeps the sums below it; -1 if no element weighs anything.
template <bool VEC>
__device__ __forceinline__ int segment_find(const Rows& r, int lo, int hi, double base, double point, int lane) {
  int last = -1;
  for (int v0 = lo; v0 < hi; v0 += 128) {
    const int v = v0 + 4 * lane;
    double w[4] = {0.0, 0.0, 0.0, 0.0};
    if (v < hi) weights4<VEC>(r, v, hi, w);
    const double mine = (w[0] + w[1]) + (w[2] + w[3]);
    const double upto = lane_scan(mine, lane);
    double c = __shfl_up_sync(0xffffffffu, upto, 1);
    c = base + (lane == 0 ? 0.0 : c);
    int hit = -1, top = -1;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c += w[j];
      if (w[j] > 0.0) { top = v + j; if (hit < 0 && c > point) hit = v + j; }
    }
    const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0);
    if (hits) return __shfl_sync(0xffffffffu, hit, __ffs(hits) - 1);
    const unsigned tops = __ballot_sync(0xffffffffu, top >= 0);
    if (tops) last = __shfl_sync(0xffffffffu, top, 31 - __clz(tops));
    base += __shfl_sync(0xffffffffu, upto, 31);
  }
  return last;
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads, 4) verify_draft_kernel(const float* target, long long target_stride,
                                                                const float* draft, long long draft_stride,
                                                                const long long* ids, const float* u,
                                                                int* accepted, long long* tokens, int S, int V,
                                                                int slice) {
  __shared__ double s_sum[kSegs];
  __shared__ double s_all[kMaxCluster * kSegs];
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank(), b = blockIdx.x / ranks;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  k3g::follow_launch();

  // every warp decides for itself which drafts stay
  bool valid = false, keep = false;
  if (lane < S) {
    const long long x = k3g::ld_ordered(ids + (long long)b * S + lane);
    valid = x >= 0 && x < V;
    if (valid) {
      const double px = k3g::ld_ordered(target + ((long long)b * (S + 1) + lane) * target_stride + x);
      const double qx = draft ? (double)k3g::ld_ordered(draft + ((long long)b * S + lane) * draft_stride + x) : 1.0;
      keep = (double)k3g::ld_ordered(u + (long long)b * (S + 1) + lane) * qx < px;
    }
  }
  const unsigned kept_mask = __ballot_sync(0xffffffffu, valid && keep), valid_mask = __ballot_sync(0xffffffffu, valid);
  const int kept = __ffs(~kept_mask) ? min(__ffs(~kept_mask) - 1, S) : S;
  const bool turned_down = kept < S && ((valid_mask >> kept) & 1u);
  Rows r;
  r.p = target + ((long long)b * (S + 1) + kept) * target_stride;
  r.q = turned_down && draft ? draft + ((long long)b * S + kept) * draft_stride : nullptr;
  r.hot = turned_down && !draft ? (int)k3g::ld_ordered(ids + (long long)b * S + kept) : -1;

  // the slice of this block, one contiguous segment (a multiple of 4 elements) for each warp
  const int seg = (slice / kSegs);
  const int lo = min(V, (rank * kSegs + warp) * seg), hi = min(V, lo + seg);
  double total = 0.0, upto = 0.0, part[4];                   // lane l looks after segments 4 l .. 4 l + 3
  for (int pass = 0; pass < 2; ++pass) {
    const double mine = segment_sum<VEC>(r, lo, hi, lane);
    if (lane == 0) s_sum[warp] = mine;
    cluster.sync();
    if (threadIdx.x < ranks * kSegs) s_all[threadIdx.x] = cluster.map_shared_rank(s_sum, threadIdx.x / kSegs)[threadIdx.x % kSegs];
    cluster.sync();                                          // read by all before any block goes on (or ends)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[j] = 4 * lane + j < ranks * kSegs ? s_all[4 * lane + j] : 0.0;
    upto = lane_scan((part[0] + part[1]) + (part[2] + part[3]), lane);
    total = __shfl_sync(0xffffffffu, upto, 31);
    if (total > 0.0 || (!r.q && r.hot < 0)) break;
    r.q = nullptr; r.hot = -1;                               // p <= q everywhere: draw from p
  }
  // the segment that holds the point: the first whose running sum passes it, else the last that weighs anything
  const double point = (double)k3g::ld_ordered(u + (long long)b * (S + 1) + S) * total;
  double base;
  const int pick_seg = part_of(part, upto, point, lane, base);
  if (rank != (pick_seg < 0 ? 0 : pick_seg / kSegs)) return;
  int pick = -1;
  bool mine = warp == 0;
  if (pick_seg >= 0) {                                       // the same once more within the segment: a part of it for each warp
    const int first = min(V, pick_seg * seg), last = min(V, first + seg), step = (seg / kSegs + 3) / 4 * 4;
    const int from = min(last, first + warp * step), to = warp == kSegs - 1 ? last : min(last, from + step);
    const double x = segment_sum<VEC>(r, from, to, lane);
    if (lane == 0) s_sum[warp] = x;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) part[j] = 4 * lane + j < kSegs ? s_sum[4 * lane + j] : 0.0;
    upto = base + lane_scan((part[0] + part[1]) + (part[2] + part[3]), lane);
    double sub_base;
    const int sub = part_of(part, upto, point, lane, sub_base, base);
    mine = warp == max(sub, 0);
    if (mine) pick = segment_find<VEC>(r, from, to, sub_base, point, lane);
  }
  if (mine) {
    if (lane == 0) accepted[b] = kept;
    for (int i = lane; i <= S; i += 32)
      tokens[(long long)b * (S + 1) + i] = i < kept ? k3g::ld_ordered(ids + (long long)b * S + i) : i == kept ? (long long)pick : -1ll;
  }
}

}  // namespace

K3G_API int k3g_verify_draft(const void* target, long long target_stride, const void* draft, long long draft_stride, const void* ids, const void* u,
                             void* accepted, void* tokens, int B, int S, int V, void* stream) {
  K3G_REQUIRE_PTR(target); K3G_REQUIRE_PTR(ids); K3G_REQUIRE_PTR(u); K3G_REQUIRE_PTR(accepted); K3G_REQUIRE_PTR(tokens);
  K3G_REQUIRE_ALIGNED(target); if (draft) K3G_REQUIRE_ALIGNED(draft);
  K3G_REQUIRE(B >= 0 && S >= 0 && V >= 0, K3G_ESHAPE);
  K3G_REQUIRE(S <= kMaxSteps && B <= (1 << 24) && V <= (1 << 30), K3G_ELIMIT);
  if (B == 0) return K3G_OK;
  K3G_REQUIRE(V > 0 && target_stride >= V && (!draft || draft_stride >= V), K3G_ESHAPE);
  // Blocks per sequence: where all blocks have an SM to themselves (148), as many as leave each 2048 elements; where they share SMs the blocks of a cluster
  // wait for one another's, and each needs 16384 to be worth it.  With 1, 2, 4 and 8 blocks a sequence, with q: 1 x 8000 entries 7.9, 6.9, 6.4, 6.4 us;
  // 1 x 163840 42, 25, 16, 10.5; 64 x 2000 5.6, 6.4, 7.4, 10.7; 64 x 8000 8.3, 7.2, 7.9, 11.2; 80 x 8000 8.4, 8.8, 10.3, 14.6; 64 x 32000 13.8, 11.0, 12.6,
  // 13.9; 80 x 32000 13.9, 15.8, 18.4, 17.3; 64 x 163840 68, 39, 28.4, 26.4; 80 x 163840 68, 46, 43, 34; 160 x 163840 83, 75, 58, 56; 296 x 163840, which two
  // blocks each just fill the card with, 87, 81, 86, 92.
  int ranks = kMaxCluster;
  while (ranks > 1 && V < ranks * ((long long)B * ranks <= 148 ? 2048 : 16384)) ranks /= 2;
  const int per = kSegs * 4 * ranks;
  const int slice = (int)(((long long)V + per - 1) / per) * kSegs * 4;
  const bool vec = target_stride % 4 == 0 && (!draft || draft_stride % 4 == 0);
  const cudaError_t e = k3g_launch_behind(vec ? verify_draft_kernel<true> : verify_draft_kernel<false>, (unsigned)(B * ranks), kThreads, 0, (unsigned)ranks,
                                          k3g_stream(stream), (const float*)target, target_stride, (const float*)draft, draft_stride, (const long long*)ids,
                                          (const float*)u, (int*)accepted, (long long*)tokens, S, V, slice);
  if (e != cudaSuccess) { cudaGetLastError(); return (int)e; }
  return k3g_launch_status();
}
