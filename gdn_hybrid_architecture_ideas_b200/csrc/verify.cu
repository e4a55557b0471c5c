// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Row b with m drafts x_0 .. x_{m-1}, target probabilities p_i (m + 1 positions) and draft probabilities q_i: draft i is
// kept while every earlier one is and u_i q_i(x_i) < p_i(x_i). Behind the kept ones comes one drawn token: at the first
// rejection i from max(p_i - q_i, 0), after the last kept draft from p_m; where that residual is zero everywhere, from p_i.
// Drawn is the first token whose running sum exceeds u * total. Without draft probabilities each draft counts as certain
// (q_i(x_i) = 1), so the residual is p_i without x_i.
//
// The comparison and the sums run in 64 bits: a product of two float32 is exact there, and running sums of 10^5 terms
// in another order differ by 1e-16 of the total, so that the token drawn does not depend on how the row was split.
//
// Only the row of probabilities that the last token is drawn from is read whole. One cluster of CTAs per row; every warp
// owns one contiguous range of the vocabulary, sums it (pass 1: all bytes of the row, once), the totals of all warps meet
// in the shared memory of every CTA of the cluster, each warp finds the range that the threshold falls into, and the one
// warp that owns it walks it again (pass 2: its range alone, from L1 / L2). No workspace, no atomics, one launch.
//
// Bound by latency: which row is read follows from three dependent loads, and each of the clusters' meetings waits for its slowest
// warp. 96 rows of 64,000 float32 probabilities with a draft's (49 MB): 16 us from L2, 26 us from memory (floor 7.5).
#include <cooperative_groups.h>

#include "paged.cuh"

namespace ghb {

namespace cg = cooperative_groups;

constexpr int VWARPS = 16;         // at most, a CTA
constexpr int VMAXCL = 8;

template <typename T> __device__ __forceinline__ double to_double(T x) { return static_cast<double>(static_cast<float>(x)); }

// The weight of a token: p, or max(p - q, 0), or p without token x. Anything not above zero (NaN too) is 0.
template <typename T>
struct Weights {
  const T* p; const T* q; int x;       // q null: no subtraction; x: the token left out, or -1
  bool wide;
  __device__ __forceinline__ double one(int j) const {
    double w = to_double(p[j]);
    if (q) w -= to_double(q[j]);
    return (w > 0.0 && j != x) ? w : 0.0;
  }
  static __device__ __forceinline__ void load4(const float* s, float* a) {
    const float4 u = *reinterpret_cast<const float4*>(s);
    a[0] = u.x; a[1] = u.y; a[2] = u.z; a[3] = u.w;
  }
  static __device__ __forceinline__ void load4(const __nv_bfloat16* s, float* a) {
    const uint2 u = *reinterpret_cast<const uint2*>(s);
    const float2 f0 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.x)), f1 = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u.y));
    a[0] = f0.x; a[1] = f0.y; a[2] = f1.x; a[3] = f1.y;
  }
};

// The lane's whole groups of four at j, j + stride, .. below hi, DEEP of them at a time: all loads of a step stand before its first sum
// and no branch between them (in place of a group behind the end the last one is read, and not counted), so that 16 bytes * DEEP * (one or two
// arrays) a lane are under way. A rest of one to three tokens is left.
template <typename T, bool Q>
__device__ __forceinline__ void wide_sum(const Weights<T>& w, int j, int hi, int stride, double& s0, double& s1) {
  constexpr int DEEP = 4;
  const int end = (hi & ~3) - 4;          // the last whole group
  for (; j <= end; j += DEEP * stride) {
    float a[DEEP][4], b[DEEP][4];
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      const int at = min(j + i * stride, end);
      w.load4(w.p + at, a[i]);
      if (Q) w.load4(w.q + at, b[i]);
    }
#pragma unroll
    for (int i = 0; i < DEEP; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const double d = Q ? static_cast<double>(a[i][c]) - static_cast<double>(b[i][c]) : static_cast<double>(a[i][c]);
        (i & 1 ? s1 : s0) += d > 0.0 && j + i * stride <= end && j + i * stride + c != w.x ? d : 0.0;
      }
  }
}
// The sum of the lane's groups (lo a multiple of four; the whole range is walked where stride is 128 and j = lo + 4 lane).
template <typename T>
__device__ __forceinline__ double lane_sum(const Weights<T>& w, int j, int hi, int stride) {
  double s0 = 0.0, s1 = 0.0;
  if (w.wide) {
    if (w.q) wide_sum<T, true>(w, j, hi, stride, s0, s1); else wide_sum<T, false>(w, j, hi, stride, s0, s1);
    const int rest = hi & ~3;                 // the vocabulary's last one to three tokens: a group that nobody read whole
    if (rest < hi && rest >= j && (rest - j) % stride == 0) for (int i = rest; i < hi; ++i) s0 += w.one(i);
  } else {
    for (; j < hi; j += stride) for (int i = j; i < min(hi, j + 4); ++i) s0 += w.one(i);
  }
  return s0 + s1;
}

template <typename T>
__device__ __forceinline__ double range_sum(const Weights<T>& w, int lo, int hi, int lane) {
  double s = lane_sum(w, lo + lane * 4, hi, 128);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// 1 / 32 of the range a lane, so that all of it is on its way at once: the lane's part that the threshold falls into, and what lies
// before it in `before`; the last part of positive weight where none does. The part is walked by range_pick.
template <typename T>
__device__ __forceinline__ void narrow(const Weights<T>& w, int& lo, int& hi, double& before, double thr, int lane) {
  const int part = ((hi - lo + 31) / 32 + 3) & ~3, l0 = min(hi, lo + lane * part), l1 = min(hi, l0 + part);
  const double s = l0 < l1 ? lane_sum(w, l0, l1, 4) : 0.0;
  double upto = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const double up = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += up; }
  double ahead = __shfl_up_sync(0xffffffffu, upto, 1);
  if (lane == 0) ahead = 0.0;
  const unsigned hits = __ballot_sync(0xffffffffu, s > 0.0 && before + upto > thr), lives = __ballot_sync(0xffffffffu, s > 0.0);
  if (!lives) return;
  const int at = hits ? __ffs(hits) - 1 : 31 - __clz(lives);
  before += __shfl_sync(0xffffffffu, ahead, at);
  lo = __shfl_sync(0xffffffffu, l0, at);
  hi = __shfl_sync(0xffffffffu, l1, at);
}

// First token of lo .. hi whose running sum, from `before` on, exceeds thr; the last one of positive weight where none does.
template <typename T>
__device__ __forceinline__ int range_pick(const Weights<T>& w, int lo, int hi, double before, double thr, int lane) {
  int live = -1;
  for (int base = lo; base < hi; base += 128) {
    const int j = base + lane * 4;
    double a[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = j + i < hi ? w.one(j + i) : 0.0;
    double run[4] = {a[0], a[0] + a[1], 0.0, 0.0};
    run[2] = run[1] + a[2]; run[3] = run[2] + a[3];
    double mine = run[3];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const double up = __shfl_up_sync(0xffffffffu, mine, o); if (lane >= o) mine += up; }
    double ahead = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == 0) ahead = 0.0;
    int hit = -1;
#pragma unroll
    for (int i = 3; i >= 0; --i) { if (a[i] > 0.0 && before + ahead + run[i] > thr) hit = j + i; }
    int last = -1;
#pragma unroll
    for (int i = 0; i < 4; ++i) if (a[i] > 0.0) last = j + i;
    const unsigned m = __ballot_sync(0xffffffffu, hit >= 0);
    if (m) return __shfl_sync(0xffffffffu, hit, __ffs(m) - 1);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    live = max(live, last);
    before += __shfl_sync(0xffffffffu, mine, 31);
  }
  return live;
}

template <typename T>
__global__ void __launch_bounds__(VWARPS * 32, 2) verify_drafts_kernel(VerifyArgs a) {
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ double totals[2][VMAXCL * VWARPS];
  __shared__ int s_kept;
  const int CL = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  cluster.barrier_arrive();              // every CTA of the cluster runs before another one writes into its shared memory
  const int b = blockIdx.x / CL;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* target = static_cast<const T*>(a.target) + b * a.t_bs;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * a.d_bs : nullptr;
  const long* drafts = a.drafts + static_cast<long>(b) * a.N;
  int m = a.n_drafts ? a.n_drafts[b] : a.N;
  if (m < 0 || m > a.N) { *a.err = ST_DRAFTS; m = m < 0 ? 0 : a.N; }
  if (warp == 0) {
    int kept = m;
    for (int i0 = 0; i0 < m; i0 += 32) {
      const int i = i0 + lane;
      bool ok = false;
      if (i < m) {
        const long x = drafts[i];
        if (x < 0 || x >= a.V) *a.err = ST_TOKEN;
        else {
          const double q = draft ? to_double(draft[i * a.d_ns + x]) : 1.0;
          ok = static_cast<double>(a.u_accept[static_cast<long>(b) * a.N + i]) * q < to_double(target[i * a.t_ns + x]);
        }
      }
      const unsigned no = __ballot_sync(0xffffffffu, i < m && !ok);
      if (no) { kept = i0 + __ffs(no) - 1; break; }
    }
    if (lane == 0) s_kept = kept;
  }
  __syncthreads();
  const int kept = s_kept;
  const bool refused = kept < m;
  Weights<T> w;
  w.p = target + kept * a.t_ns;
  w.q = refused && draft ? draft + kept * a.d_ns : nullptr;
  w.x = refused && !draft ? static_cast<int>(drafts[kept] >= 0 && drafts[kept] < a.V ? drafts[kept] : -1) : -1;
  w.wide = (reinterpret_cast<uintptr_t>(w.p) | reinterpret_cast<uintptr_t>(w.q)) % (4 * sizeof(T)) == 0 && a.V >= 4;
  const int warps = static_cast<int>(blockDim.x) >> 5, ranges = CL * warps, mine = rank * warps + warp;
  const int per = ((a.V + ranges - 1) / ranges + 3) & ~3;
  const int lo = min(a.V, mine * per), hi = min(a.V, lo + per);
  double total = 0.0, t4[4], ahead = 0.0;
  int phase = 0;
  for (; phase < 2; ++phase) {
    const double s = range_sum(w, lo, hi, lane);
    if (phase == 0) cluster.barrier_wait();
    if (lane < CL) *cluster.map_shared_rank(&totals[phase][mine], lane) = s;
    cluster.sync();
    // four ranges a lane (there are at most 128): their sums, and by a scan over the lanes what lies before them
    double mine4 = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) { t4[i] = 4 * lane + i < ranges ? totals[phase][4 * lane + i] : 0.0; mine4 += t4[i]; }
    double upto = mine4;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const double up = __shfl_up_sync(0xffffffffu, upto, o); if (lane >= o) upto += up; }
    ahead = __shfl_up_sync(0xffffffffu, upto, 1);
    if (lane == 0) ahead = 0.0;
    total = __shfl_sync(0xffffffffu, upto, 31);
    if (total > 0.0 || !refused) break;
    w.q = nullptr; w.x = -1;             // the residual is zero everywhere: the target itself (every CTA sees the same totals)
  }
  // the first range at whose end the running sum exceeds the threshold (every warp finds the same); the last one of positive weight
  // where rounding leaves none
  const double thr = static_cast<double>(a.u_sample[b]) * total;
  int owner = ranges, last = -1;
  double before = 0.0, before_last = 0.0, run = ahead;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (t4[i] > 0.0) { last = 4 * lane + i; before_last = run; }
    if (owner == ranges && run + t4[i] > thr) { owner = 4 * lane + i; before = run; }
    run += t4[i];
  }
  const unsigned hits = __ballot_sync(0xffffffffu, owner < ranges), lives = __ballot_sync(0xffffffffu, last >= 0);
  if (hits) {
    owner = __shfl_sync(0xffffffffu, owner, __ffs(hits) - 1);
    before = __shfl_sync(0xffffffffu, before, __ffs(hits) - 1);
  } else if (lives) {
    owner = __shfl_sync(0xffffffffu, last, 31 - __clz(lives));
    before = __shfl_sync(0xffffffffu, before_last, 31 - __clz(lives));
  } else {
    owner = -1;
  }
  long* out = a.tokens + static_cast<long>(b) * (a.N + 1);
  if (owner == mine) {
    int from = lo, to = hi;
    narrow(w, from, to, before, thr, lane);
    const int pick = range_pick(w, from, to, before, thr, lane);
    if (lane == 0) out[kept] = pick < 0 ? 0 : pick;
  }
  if (rank == 0) {
    for (int i = threadIdx.x; i <= a.N; i += blockDim.x)
      if (i != kept) out[i] = i < kept ? drafts[i] : -1;
    if (threadIdx.x == 0) {
      a.kept[b] = kept;
      if (owner < 0) out[kept] = 0;      // a row without any positive probability
    }
  }
}

int verify_drafts(const VerifyArgs& a, cudaStream_t st) {
  if (a.B == 0) return 0;
  if (a.V < 1 || a.N < 0 || a.B > 0x7fffffff / VMAXCL) return 1;
  // CTAs a row: 8, 4 or 2 of 8 warps, as long as the grid leaves an eighth of the GPU's places (4 such CTAs an SM) free: whole clusters
  // wait for places in one GPC. Two of 16 warps where those still are one wave. Measured at 64,000 float32 probabilities with a
  // draft's, 8 / 4 / 2 CTAs of 8 warps, 2 of 16: 24 rows 8.2 / 9.8 / 14.4, 11.1 us; 96 rows 17.3 / 14.6 / 19.8, 16.6 us;
  // 148 rows 24.4 / 22.4 / 22.2, 18.5 us; 600 rows 74 / 58 / 56, 64 us. Cluster sizes that are no powers of two were slower than both
  // neighbours. A warp has 128 probabilities at least.
  int cl = VMAXCL, warps = VWARPS / 2;
  while (cl > 2 && static_cast<long>(a.B) * cl > 148 * 7 / 2) cl >>= 1;
  if (cl == 2 && a.B <= 148) warps = VWARPS;
  while (cl > 1 && a.V < 128 * warps * cl) cl >>= 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.B * cl);
  cfg.blockDim = dim3(warps * 32);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  const cudaError_t rc = a.bf16 ? cudaLaunchKernelEx(&cfg, verify_drafts_kernel<__nv_bfloat16>, a) : cudaLaunchKernelEx(&cfg, verify_drafts_kernel<float>, a);
  return rc == cudaSuccess ? 0 : 4;
}

}  // namespace ghb
