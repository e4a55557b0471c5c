// Attention of one or a few new tokens a row over a paged key/value cache in bfloat16 or 4 bits (layout and checks:
// paged.cuh). Query row r of a (batch row, KV head): new token r / G, head r % G of the group; it sees the cached positions
// from the row's start up to its own. Scores: q rotated at its position . k (cached rotated); under a rotary distance
// cap C the cache holds the keys unrotated and R(p_q) q . R(p_k) k counts up to distance C, R(C) q . k beyond it.
//
// Products run transposed on mma.sync m16n8k16: S^T = K Q^T with 16 cached positions as rows and 8 query rows as columns, and
// O^T = V^T P^T with 16 channels as rows. A decode step has G (4 or 8) query rows for each KV head, so the transposed form
// fills the tile, where query rows as the 16-high side would leave three quarters of it empty; tcgen05's 128-row
// tile would be 97% empty, and its block-scaled 4-bit kind would need 4-bit queries and probabilities. S^T's accumulator
// layout and P^T's operand layout differ by an 8 x 8 transposition (movmatrix); columns (query rows) stay in their lanes, so
// the softmax's running maximum and sum are registers, and only the maximum needs shuffles (over the 8 lane groups).
//
// 4 bits: a lane's 16 channels of a key are one block with one scale. Codes become f16 pairs (cvt.f16x2.e2m1x2), times the
// scale: exact in f16 (2 + 4 significant bits, 2^-10 .. 2688). Queries are rounded to f16 once (2^-12 relative), after a
// power of two per query row has brought them to about one, probabilities to f16 scaled by 2^14, so that one of 2^-28 of the
// maximum is still normal. bfloat16 cache: queries as the sum of two bfloat16 (2^-17), keys as they are, probabilities to
// bfloat16 (2^-9) with the sum taken over the rounded ones. All sums are float32 in the accumulators.
//
// Work: the pieces (one tile of positions for each warp) of all (row, KV head, block of query rows) units form one sequence,
// and every CTA takes an equal share of it, so that rows of any lengths load the SMs evenly. Each CTA finds its share by
// a prefix sum over the rows. Warps take the tiles of a piece and keep their own running softmax; they meet in shared memory at
// the end of a unit's part. A unit cut by CTA borders leaves partial results (at most two a CTA), joined by a second kernel in
// the order of the CTAs: no atomics, the same result every time.
//
// Loads: cp.async into a ring of tiles private to each warp (no block barrier in the loop); what is not visible
// (before the start, behind the length, under a bad page id) is not read but filled with zeros.
#include "paged.cuh"

namespace ghb {

struct AttnK {                       // by value to the kernels
  PagedRows r; PagedPool c; PagedAttn a;
  int G;
  float* ws; int* meta;
};

template <bool FP4, int HD> struct Cfg;
template <> struct Cfg<true, 64> { static constexpr int W = 8, ST = 4, CTAS = 2; };
template <> struct Cfg<true, 128> { static constexpr int W = 8, ST = 3, CTAS = 2; };
template <> struct Cfg<true, 256> { static constexpr int W = 4, ST = 3, CTAS = 2; };
template <> struct Cfg<false, 64> { static constexpr int W = 8, ST = 3, CTAS = 2; };
template <> struct Cfg<false, 128> { static constexpr int W = 4, ST = 3, CTAS = 2; };
template <> struct Cfg<false, 256> { static constexpr int W = 4, ST = 3, CTAS = 1; };

template <bool FP4, int HD, int NT>
struct Geo : Cfg<FP4, HD> {
  using B = Cfg<FP4, HD>;
  static constexpr int MT = FP4 ? 2 : 1;             // 16-position tiles a warp takes at once
  static constexpr int TILE = 16 * MT;
  static constexpr int H = HD / 64;                  // 64-channel slices
  static constexpr int KB = FP4 ? TILE * HD / 2 : TILE * HD * 2;      // bytes of a tile's keys (values the same)
  static constexpr int SB = FP4 ? TILE * HD / 16 : 0;                 // bytes of its scales
  static constexpr int STAGE = 2 * KB + 2 * SB;
  static constexpr int UR = 8 * NT;                  // query rows of a unit
  static constexpr int PIECE = B::W * TILE;
  static constexpr int RING = B::W * B::ST * STAGE;
  static constexpr int MERGE = B::W * UR * HD * 4;
  static constexpr int DATA = RING > MERGE ? RING : MERGE;
  static constexpr int QCOPIES = FP4 ? 1 : 2;        // bfloat16: high and low part
  static constexpr int QB = UR * HD * 2;             // bytes of one copy of the queries
  static constexpr int SMEM = DATA + 2 * QCOPIES * QB;       // near and far queries
  static constexpr int THREADS = B::W * 32;
};

constexpr float PSHIFT = 14.f;

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
template <int BYTES>
__device__ __forceinline__ void cp_small(uint32_t dst, const void* src, bool on) {
  if constexpr (BYTES == 16) cp16(dst, src, on);
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %3, %2;" ::"r"(dst), "l"(src), "r"(on ? BYTES : 0), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool FP4>
__device__ __forceinline__ void mma(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (FP4)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float exp2_fast(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// eight codes (a 32-bit word) -> four f16 pairs
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t* h) {
  asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\tmov.b32 {c0, c1, c2, c3}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, c0;\n\tcvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c2;\n\tcvt.rn.f16x2.e2m1x2 %3, c3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
// two E4M3 scales (bytes 0 and 1) -> an f16 pair
__device__ __forceinline__ uint32_t scales_to_f16(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 c;\n\tcvt.u16.u32 c, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(two));
  return h;
}
template <bool FP4>
__device__ __forceinline__ float2 unpack(uint32_t x) {
  if constexpr (FP4) return __half22float2(*reinterpret_cast<const __half2*>(&x));
  else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x));
}
template <bool FP4>
__device__ __forceinline__ uint32_t pack(float a, float b) {
  if constexpr (FP4) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
  else { const __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<const uint32_t*>(&h); }
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Row rho (0 .. 7) of an 8-row group of the tiles is position place(rho) of the group. 4 bits: chosen so that both the keys' reads
// (8 bytes of rows rho = 0..3 or 4..7 at once) and the values' (4 bytes of rows 0,2,4,6 or 1,3,5,7) touch four
// 32-byte rows that differ modulo 4, hence all 32 banks. bfloat16 rows are 128 bytes and swizzled by 16-byte chunk instead.
template <bool FP4> __device__ __forceinline__ int place(int rho) {
  return FP4 ? (rho & 4) | (((rho ^ (rho >> 2)) & 1) << 1) | ((rho >> 1) & 1) : rho;
}

// The units of a row: how many for a head, and how many pieces each.
struct RowWork { int units, pieces, base; };
template <typename GEO>
__device__ __forceinline__ RowWork row_work(const Row& row, int G) {
  RowWork w;
  w.units = (row.nq * G + GEO::UR - 1) / GEO::UR;
  w.base = row.start & ~(GEO::TILE - 1);
  const int span = row.len - w.base;
  w.pieces = span > 0 ? (span + GEO::PIECE - 1) / GEO::PIECE : 1;      // a row that sees nothing still owes zeros
  return w;
}

template <int THREADS>
__device__ __forceinline__ long block_scan(long x, long* s_warp, long* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  long inc = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const long up = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += up; }
  __syncthreads();
  if (lane == 31) s_warp[warp] = inc;
  __syncthreads();
  long before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) { if (w < warp) before += s_warp[w]; all += s_warp[w]; }
  *total = all;
  return before + inc - x;      // exclusive
}

template <bool FP4, int HD, int NT>
__global__ void __launch_bounds__(Geo<FP4, HD, NT>::THREADS, Geo<FP4, HD, NT>::CTAS) paged_attention_kernel(const __grid_constant__ AttnK p) {
  using GEO = Geo<FP4, HD, NT>;
  constexpr int H = GEO::H, MT = GEO::MT, TILE = GEO::TILE, UR = GEO::UR, W = GEO::W, ST = GEO::ST;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long s_warp[W];
  __shared__ long s_at[2];
  __shared__ float s_mul[UR];                 // a query row's factor on its scores: scale * log2(e) * its power of two
  __shared__ float s_m[W][UR], s_l[W][UR];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const PagedRows& R = p.r;
  const int n_ctas = gridDim.x, cta = blockIdx.x, Hkv = R.Hkv, G = p.G;

  // ---- this CTA's share of the pieces
  long total = 0;
  if (tid < 2) s_at[tid] = -1;
  for (int b0 = 0; b0 < R.B; b0 += GEO::THREADS) {
    long mine = 0, all;
    if (b0 + tid < R.B) { const RowWork w = row_work<GEO>(load_row(R, b0 + tid), G); mine = static_cast<long>(w.units) * w.pieces * Hkv; }
    block_scan<GEO::THREADS>(mine, s_warp, &all);
    total += all;
  }
  const long use = total < n_ctas ? total : n_ctas;      // CTAs with work: at least one piece each
  int* meta = p.meta + cta * 8;
  if (cta >= use) {
    if (tid < 2) meta[tid * 4] = -1;
    return;
  }
  const long lo = total * cta / use, hi = total * (cta + 1) / use;
  {
    long before = 0;
    for (int b0 = 0; b0 < R.B; b0 += GEO::THREADS) {
      long mine = 0, all;
      if (b0 + tid < R.B) { const RowWork w = row_work<GEO>(load_row(R, b0 + tid), G); mine = static_cast<long>(w.units) * w.pieces * Hkv; }
      const long ex = before + block_scan<GEO::THREADS>(mine, s_warp, &all);
      if (lo >= ex && lo < ex + mine) { s_at[0] = b0 + tid; s_at[1] = ex; }
      before += all;
      if (before > lo) break;
    }
  }
  __syncthreads();
  int b = static_cast<int>(s_at[0]);
  long row_at = s_at[1];
  if (tid < 2) meta[tid * 4] = -1;
  __syncthreads();

  uint8_t* ring = smem + warp * (ST * GEO::STAGE);
  const uint32_t ring_u = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  uint8_t* sq = smem + GEO::DATA;

  long at = lo;
  while (at < hi) {
    // ---- the unit that piece `at` belongs to
    Row row = load_row(R, b);
    RowWork wk = row_work<GEO>(row, G);
    long count = static_cast<long>(wk.units) * wk.pieces * Hkv;
    while (at >= row_at + count) {            // rows without tokens have no pieces
      row_at += count;
      ++b;
      row = load_row(R, b);
      wk = row_work<GEO>(row, G);
      count = static_cast<long>(wk.units) * wk.pieces * Hkv;
    }
    const long in_row = at - row_at;
    const int unit = static_cast<int>(in_row / wk.pieces), p0 = static_cast<int>(in_row % wk.pieces);
    const int n_pieces = static_cast<int>(min(static_cast<long>(wk.pieces - p0), hi - at));
    const int h = unit / wk.units, r0 = (unit % wk.units) * UR;
    const int n_rows = min(UR, row.nq * G - r0);
    const int pos0 = row.len - row.nq;                              // position of the row's first new token
    const int p_first = pos0 + r0 / G, p_last = row.len ? pos0 + (r0 + n_rows - 1) / G : -1;
    // ---- loads of one tile: positions base .. base + TILE
    const int tile0 = wk.base + p0 * GEO::PIECE + warp * TILE;
    auto page_at = [&](int k) -> int {         // page id of this lane's position of tile k, -1: not read
      const int tok = tile0 + k * GEO::PIECE + (lane & (TILE - 1));
      if (k >= n_pieces || tok < row.start || tok > p_last) return -1;
      const int pg = R.pages[b * R.pages_stride + (tok >> R.page_shift)];
      if (pg < 0 || pg >= R.n_pages) { *R.err = ST_PAGE; return -1; }
      return pg;
    };
    auto issue = [&](int k, int pg) -> unsigned {      // returns the mask of positions that are read
      const int tok = tile0 + k * GEO::PIECE + (lane & (TILE - 1));
      const unsigned on = __ballot_sync(0xffffffffu, pg >= 0);
      if (k < n_pieces) {
        const uint32_t st = ring_u + (k % ST) * GEO::STAGE;
        const int e = pg >= 0 ? ((pg * Hkv + h) << R.page_shift) + (tok & ((1 << R.page_shift) - 1)) : 0;
        constexpr int ROW = FP4 ? HD / 2 : HD * 2, CH = ROW / 16;      // bytes and 16-byte chunks of a position
        const uint8_t* kb = static_cast<const uint8_t*>(p.c.k);
        const uint8_t* vb = static_cast<const uint8_t*>(p.c.v);
#pragma unroll
        for (int i = 0; i < TILE * CH / 32; ++i) {
          const int idx = i * 32 + lane, pos = idx / CH, sub = idx % CH;
          const int ee = __shfl_sync(0xffffffffu, e, pos);
          const bool ok = (on >> pos) & 1;
          uint32_t dst;
          if constexpr (FP4) dst = (sub >> 1) * (TILE * 32) + pos * 32 + (sub & 1) * 16;
          else dst = (sub >> 3) * (TILE * 128) + pos * 128 + (((sub & 7) ^ (pos & 7)) << 4);
          const long off = static_cast<long>(ee) * ROW + sub * 16;
          cp16(st + dst, kb + off, ok);
          cp16(st + GEO::KB + dst, vb + off, ok);
        }
        if constexpr (FP4) {
          constexpr int S = HD / 16;
          const long off = static_cast<long>(e) * S;
          cp_small<S>(st + 2 * GEO::KB + lane * S, p.c.k_scale + off, pg >= 0);
          cp_small<S>(st + 2 * GEO::KB + GEO::SB + lane * S, p.c.v_scale + off, pg >= 0);
        }
      }
      cp_commit();
      return on;
    };
    unsigned on_ring[ST];
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) on_ring[k] = issue(k, page_at(k));
    int pg_next = page_at(ST - 1);

    // ---- the unit's queries: rotated (near at their positions, far by the cap), brought to about one, in the MMA's order
    for (int r = warp; r < UR; r += W) {
      const bool live = r < n_rows && row.len > 0;
      const int rr = r0 + r;
      const long tok = row.q0 + (live ? rr / G : 0);
      const int head = h * G + (live ? rr % G : 0);
      const long off = tok * p.a.q_ts + head * p.a.q_hs;
      auto qv = [&](int c) -> float {
        return p.a.q_f32 ? static_cast<const float*>(p.a.q)[off + c] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.a.q)[off + c]);
      };
      float x[HD / 32];
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) { x[i] = live ? qv(lane + 32 * i) : 0.f; top = fmaxf(top, fabsf(x[i])); }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      int ex = 0;
      if (FP4 && top > 0.f && top < INFINITY) ex = ilogbf(top);
      ex = max(-120, min(120, ex));
      const float down = exp2f(static_cast<float>(-ex));
      if (lane == 0) s_mul[r] = p.a.scale * 1.44269504088896340736f * exp2f(static_cast<float>(ex));
      int qpos = pos0 + rr / G - row.start;
      if (live && p.a.half > 0 && qpos >= p.a.n_pos) { *R.err = ST_ROPE; qpos = p.a.n_pos - 1; }
      qpos = max(qpos, 0);
#pragma unroll
      for (int i = 0; i < HD / 32; ++i) {
        const int c = lane + 32 * i, half = p.a.half;
        float near = x[i], far = x[i];
        if (live && c < 2 * half) {
          const bool lowside = c < half;
          const int ai = lowside ? c : c - half;
          const float y = qv(lowside ? c + half : c - half), sg = lowside ? -y : y;
          near = x[i] * p.a.cos[static_cast<long>(qpos) * half + ai] + sg * p.a.sin[static_cast<long>(qpos) * half + ai];
          if (p.a.cap) far = x[i] * p.a.cos[static_cast<long>(p.a.cap) * half + ai] + sg * p.a.sin[static_cast<long>(p.a.cap) * half + ai];
        }
        const int cc = c & 63;
        const int idx = ((((r >> 3) * (HD / 16) + (c >> 6) * 4 + ((cc & 15) >> 2)) * 32 + (r & 7) * 4 + (cc >> 4)) << 2) + (cc & 3);
        if constexpr (FP4) {
          reinterpret_cast<__half*>(sq)[idx] = __float2half_rn(near * down);
          if (p.a.cap) reinterpret_cast<__half*>(sq + GEO::QB)[idx] = __float2half_rn(far * down);
        } else {
          const __nv_bfloat16 n1 = __float2bfloat16(near), f1 = __float2bfloat16(far);
          reinterpret_cast<__nv_bfloat16*>(sq)[idx] = n1;
          // (an infinite part has no remainder: inf - inf would turn it into NaN a second time, which it is in the product anyway)
          reinterpret_cast<__nv_bfloat16*>(sq + GEO::QB)[idx] = __float2bfloat16(isfinite(near) ? near - __bfloat162float(n1) : 0.f);
          if (p.a.cap) {
            reinterpret_cast<__nv_bfloat16*>(sq + 2 * GEO::QB)[idx] = f1;
            reinterpret_cast<__nv_bfloat16*>(sq + 3 * GEO::QB)[idx] = __float2bfloat16(isfinite(far) ? far - __bfloat162float(f1) : 0.f);
          }
        }
      }
    }
    __syncthreads();

    float mul[NT][2], m[NT][2], l[NT][2];
    int prow[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = n * 8 + 2 * t + e;
        mul[n][e] = s_mul[r];
        prow[n][e] = r < n_rows && row.len > 0 ? pos0 + (r0 + r) / G : -1;
        m[n][e] = -INFINITY; l[n][e] = 0.f;
      }
    float o[H * 4][NT][4];
#pragma unroll
    for (int i = 0; i < H * 4; ++i)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][n][e] = 0.f;

    for (int k = 0; k < n_pieces; ++k) {
      {
        const unsigned on = issue(k + ST - 1, pg_next);
        pg_next = page_at(k + ST);
        cp_wait<ST - 1>();
        __syncwarp();
        // the masks travel with the ring
        const unsigned now = on_ring[0];
#pragma unroll
        for (int i = 0; i < ST - 2; ++i) on_ring[i] = on_ring[i + 1];
        on_ring[ST - 2] = on;
        on_ring[ST - 1] = now;
      }
      const unsigned on = on_ring[ST - 1];
      const int first = tile0 + k * GEO::PIECE;
      if (on) {
        const uint8_t* st = ring + (k % ST) * GEO::STAGE;
        const bool far_any = p.a.cap && p_last - first > p.a.cap;                       // some (row, position) beyond the cap
        const bool near_any = !p.a.cap || p_first - (first + TILE - 1) <= p.a.cap;      // some within it
        float s[MT][NT][4];

        auto score = [&](bool rotate, const uint8_t* qs, float (&acc)[MT][NT][4]) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[mt][n][e] = 0.f;
#pragma unroll
          for (int hs = 0; hs < H; ++hs) {
            uint32_t x[MT][2][8];                // [tile][row g or g + 8][channel pair]: channels 16 t + 2 i of slice hs
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int pos = mt * 16 + e * 8 + place<FP4>(g);
                if constexpr (FP4) {
                  const uint2 w = *reinterpret_cast<const uint2*>(st + hs * (TILE * 32) + pos * 32 + t * 8);
                  uint32_t sc = st[2 * GEO::KB + pos * (HD / 16) + hs * 4 + t];
                  sc = scales_to_f16(sc | (sc << 8));
                  codes_to_f16(w.x, x[mt][e]);
                  codes_to_f16(w.y, x[mt][e] + 4);
#pragma unroll
                  for (int i = 0; i < 8; ++i) x[mt][e][i] = hmul2(x[mt][e][i], sc);
                } else {
#pragma unroll
                  for (int c = 0; c < 2; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4*>(st + hs * (TILE * 128) + pos * 128 + (((2 * t + c) ^ (pos & 7)) << 4));
                    x[mt][e][4 * c] = w.x; x[mt][e][4 * c + 1] = w.y; x[mt][e][4 * c + 2] = w.z; x[mt][e][4 * c + 3] = w.w;
                  }
                }
              }
            if (hs == 0 && rotate) {
              // channel i < half with i + half: both in this lane (half 8), or in the lane half / 16 away
              const int half = p.a.half;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int tok = first + mt * 16 + e * 8 + place<FP4>(g);
                  const int pp = max(0, min(tok - row.start, p.a.n_pos - 1));
                  const float* co = p.a.cos + static_cast<long>(pp) * half;
                  const float* si = p.a.sin + static_cast<long>(pp) * half;
                  uint32_t* y = x[mt][e];
                  if (half == 8) {
                    if (t == 0) {
#pragma unroll
                      for (int i = 0; i < 4; ++i) {
                        const float2 a = unpack<FP4>(y[i]), bb = unpack<FP4>(y[i + 4]);
                        const float2 c = *reinterpret_cast<const float2*>(co + 2 * i), sn = *reinterpret_cast<const float2*>(si + 2 * i);
                        y[i] = pack<FP4>(a.x * c.x - bb.x * sn.x, a.y * c.y - bb.y * sn.y);
                        y[i + 4] = pack<FP4>(bb.x * c.x + a.x * sn.x, bb.y * c.y + a.y * sn.y);
                      }
                    }
                  } else {
                    const int away = half >> 4;            // 1 or 2 lanes
                    const int base = (t & (away - 1)) * 16;
                    const bool lowside = (t & away) == 0, mine = t * 16 < 2 * half;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                      const uint32_t other = __shfl_xor_sync(0xffffffffu, y[i], away);
                      if (mine) {
                        const float2 a = unpack<FP4>(y[i]), bb = unpack<FP4>(other);
                        const float2 c = *reinterpret_cast<const float2*>(co + base + 2 * i), sn = *reinterpret_cast<const float2*>(si + base + 2 * i);
                        const float sx = lowside ? -sn.x : sn.x, sy = lowside ? -sn.y : sn.y;
                        y[i] = pack<FP4>(a.x * c.x + bb.x * sx, a.y * c.y + bb.y * sy);
                      }
                    }
                  }
                }
            }
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const int qi = ((n * (HD / 16) + hs * 4 + ks) * 32 + lane) * 8;
                const uint2 q1 = *reinterpret_cast<const uint2*>(qs + qi);
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const uint32_t a[4] = {x[mt][0][2 * ks], x[mt][1][2 * ks], x[mt][0][2 * ks + 1], x[mt][1][2 * ks + 1]};
                  mma<FP4>(acc[mt][n], a, q1.x, q1.y);
                }
                if constexpr (!FP4) {
                  const uint2 q2 = *reinterpret_cast<const uint2*>(qs + GEO::QB + qi);
#pragma unroll
                  for (int mt = 0; mt < MT; ++mt) {
                    const uint32_t a[4] = {x[mt][0][2 * ks], x[mt][1][2 * ks], x[mt][0][2 * ks + 1], x[mt][1][2 * ks + 1]};
                    mma<FP4>(acc[mt][n], a, q2.x, q2.y);
                  }
                }
              }
          }
        };
        if (near_any) score(p.a.cap != 0, sq, s);
        if (far_any) {
          const uint8_t* qf = sq + GEO::QCOPIES * GEO::QB;
          if (!near_any) score(false, qf, s);
          else {
            float sf[MT][NT][4];
            score(false, qf, sf);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int tok = first + mt * 16 + (e >> 1) * 8 + place<FP4>(g);
                  if (prow[n][e & 1] - tok > p.a.cap) s[mt][n][e] = sf[mt][n][e];
                }
          }
        }
        // ---- masks, where any (row, position) of the tile is not visible
        const unsigned whole = TILE == 32 ? 0xffffffffu : 0xffffu;
        const bool masked = (on & whole) != whole || first + TILE - 1 > p_first;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s[mt][n][e] *= mul[n][e & 1];
              if (masked) {
                const int pos = mt * 16 + (e >> 1) * 8 + place<FP4>(g);
                if (!((on >> pos) & 1) || first + pos > prow[n][e & 1]) s[mt][n][e] = -INFINITY;
              }
            }
        // ---- running maximum, probabilities
        uint32_t pk[MT][NT][2];
        float alpha[NT][2];
        bool grew = false;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = s[0][n][e];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) mx = fmaxf(mx, fmaxf(s[mt][n][e], s[mt][n][e + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float mn = fmaxf(m[n][e], mx);
            const float ref = mn == -INFINITY ? 0.f : mn;
            alpha[n][e] = exp2_fast(m[n][e] - ref);
            grew |= mn != m[n][e];
            m[n][e] = mn;
            float sum = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float pr = exp2_fast(s[mt][n][e + 2 * q] - ref + (FP4 ? PSHIFT : 0.f));
                s[mt][n][e + 2 * q] = pr;
                if constexpr (FP4) sum += pr;
              }
            if constexpr (FP4) l[n][e] = l[n][e] * alpha[n][e] + sum;
          }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q) pk[mt][n][q] = pack<FP4>(s[mt][n][2 * q], s[mt][n][2 * q + 1]);
        if constexpr (!FP4) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                const float2 f = unpack<FP4>(pk[mt][n][q]);
                s0 += f.x; s1 += f.y;
                s[mt][n][2 * q] = f.x; s[mt][n][2 * q + 1] = f.y;
              }
            l[n][0] = l[n][0] * alpha[n][0] + s0;
            l[n][1] = l[n][1] * alpha[n][1] + s1;
          }
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int i = 0; i < H * 4; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              o[i][n][0] *= alpha[n][0]; o[i][n][1] *= alpha[n][1];
              o[i][n][2] *= alpha[n][0]; o[i][n][3] *= alpha[n][1];
            }
        }
        // ---- O^T += V^T P^T
        bool plain = true;
        if constexpr (!FP4) {
          // A masked position's value may be infinite or NaN, and 0 times it would reach rows that do not see it: such a
          // tile is summed position by position, each row over what it sees.
          if (masked) {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < TILE * HD * 2 / 512; ++i) {
              const uint4 w = *reinterpret_cast<const uint4*>(st + GEO::KB + (i * 32 + lane) * 16);
              const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
              for (int c = 0; c < 4; ++c) odd |= (ws[c] & 0x7f80u) == 0x7f80u || (ws[c] & 0x7f800000u) == 0x7f800000u;
            }
            plain = !__any_sync(0xffffffffu, odd);
          }
          if (!plain) {
            for (int j = 0; j < TILE; ++j) {
              if (!((on >> j) & 1)) continue;
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                const float p0 = __shfl_sync(0xffffffffu, j < 8 ? s[0][n][0] : s[0][n][2], (j & 7) * 4 + t);
                const float p1 = __shfl_sync(0xffffffffu, j < 8 ? s[0][n][1] : s[0][n][3], (j & 7) * 4 + t);
                const bool see0 = first + j <= prow[n][0], see1 = first + j <= prow[n][1];
#pragma unroll
                for (int hs = 0; hs < H; ++hs) {
                  const uint4 w = *reinterpret_cast<const uint4*>(st + GEO::KB + hs * (TILE * 128) + j * 128 + ((g ^ (j & 7)) << 4));
                  const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                  for (int i = 0; i < 4; ++i) {
                    const float2 v = unpack<FP4>(ws[i]);
                    float* oo = o[hs * 4 + i][n];
                    if (see0) { oo[0] += p0 * v.x; oo[2] += p0 * v.y; }
                    if (see1) { oo[1] += p1 * v.x; oo[3] += p1 * v.y; }
                  }
                }
              }
            }
          }
        }
        if (plain) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) { pb[n][0] = transpose8(pk[mt][n][0]); pb[n][1] = transpose8(pk[mt][n][1]); }
            const int u0 = mt * 16 + place<FP4>(2 * t), u1 = mt * 16 + place<FP4>(2 * t + 1);
#pragma unroll
            for (int hs = 0; hs < H; ++hs) {
              uint32_t v[4][4];                    // [position u0, u1, u0 + 8, u1 + 8][channel pair 8 g + 2 i]
              uint32_t sc[2];
              if constexpr (FP4) {
                const uint8_t* vb = st + GEO::KB + hs * (TILE * 32) + g * 4;
                codes_to_f16(*reinterpret_cast<const uint32_t*>(vb + u0 * 32), v[0]);
                codes_to_f16(*reinterpret_cast<const uint32_t*>(vb + u1 * 32), v[1]);
                codes_to_f16(*reinterpret_cast<const uint32_t*>(vb + (u0 + 8) * 32), v[2]);
                codes_to_f16(*reinterpret_cast<const uint32_t*>(vb + (u1 + 8) * 32), v[3]);
                const uint8_t* sb = st + 2 * GEO::KB + GEO::SB + hs * 4 + (g >> 1);
                constexpr int S = HD / 16;
                sc[0] = scales_to_f16(static_cast<uint32_t>(sb[u0 * S]) | (static_cast<uint32_t>(sb[u1 * S]) << 8));
                sc[1] = scales_to_f16(static_cast<uint32_t>(sb[(u0 + 8) * S]) | (static_cast<uint32_t>(sb[(u1 + 8) * S]) << 8));
              } else {
                const uint8_t* vb = st + GEO::KB + hs * (TILE * 128);
                const int us[4] = {u0, u1, u0 + 8, u1 + 8};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const uint4 w = *reinterpret_cast<const uint4*>(vb + us[c] * 128 + ((g ^ (us[c] & 7)) << 4));
                  v[c][0] = w.x; v[c][1] = w.y; v[c][2] = w.z; v[c][3] = w.w;
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                uint32_t a[4] = {prmt(v[0][i], v[1][i], 0x5410), prmt(v[0][i], v[1][i], 0x7632), prmt(v[2][i], v[3][i], 0x5410), prmt(v[2][i], v[3][i], 0x7632)};
                if constexpr (FP4) { a[0] = hmul2(a[0], sc[0]); a[1] = hmul2(a[1], sc[0]); a[2] = hmul2(a[2], sc[1]); a[3] = hmul2(a[3], sc[1]); }
#pragma unroll
                for (int n = 0; n < NT; ++n) mma<FP4>(o[hs * 4 + i][n], a, pb[n][0], pb[n][1]);
              }
            }
          }
        }
      }
      __syncwarp();          // the stage is consumed before the next issue refills it
    }
    cp_wait<0>();
    __syncthreads();         // every warp is done with its ring: the region takes the partial outputs

    // ---- join the warps
    float* so = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum = l[n][e];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        const int r = n * 8 + 2 * t + e;
        if (g == 0) { s_m[warp][r] = m[n][e]; s_l[warp][r] = sum; }
        float* dst = so + (static_cast<long>(warp) * UR + r) * HD + 8 * g;
#pragma unroll
        for (int i = 0; i < H * 4; ++i)
          *reinterpret_cast<float2*>(dst + (i >> 2) * 64 + (i & 3) * 2) = make_float2(o[i][n][e], o[i][n][e + 2]);
      }
    __syncthreads();
    const bool begins = p0 == 0, ends = p0 + n_pieces == wk.pieces;
    const int slot = begins ? 1 : 0;
    float* wo = p.ws + (static_cast<long>(cta) * 2 + slot) * UR * (HD + 2);
    for (int idx = tid; idx < n_rows * HD; idx += GEO::THREADS) {
      const int r = idx / HD, c = idx % HD;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_m[w][r]);
      const float ref = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f, oo = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float f = exp2_fast(s_m[w][r] - ref);
        ll += s_l[w][r] * f;
        // (a warp that saw nothing holds zeros)
        oo += so[(static_cast<long>(w) * UR + r) * HD + c] * f;
      }
      if (begins && ends) {
        const int rr = r0 + r;
        // a row of scores without one above -inf has no weights: zeros
        static_cast<__nv_bfloat16*>(p.a.out)[((static_cast<long>(row.q0) + rr / G) * p.a.Hq + h * G + rr % G) * HD + c] = __float2bfloat16(ll == 0.f ? 0.f : oo / ll);
      } else {
        wo[r * HD + c] = oo;
        if (c == 0) { wo[UR * HD + 2 * r] = mm; wo[UR * HD + 2 * r + 1] = ll; }
      }
    }
    if (tid == 0 && !(begins && ends)) {
      int* mt = meta + slot * 4;
      mt[1] = h; mt[2] = r0; mt[3] = ends ? 1 : 0;
      mt[0] = b;
    }
    at += n_pieces;
    __syncthreads();
  }
}

// Joins the parts of every unit that CTA borders cut: part one is the last thing its first CTA did (slot 1), the others the first
// thing the following CTAs did (slot 0). Block (i, r) joins query row r of the unit whose first part CTA i holds. Also the zeros of
// the packed tokens behind the last row, where the output is this call's own.
template <int HD, int UR>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const __grid_constant__ AttnK p, int n_ctas) {
  constexpr int LANES = HD / 4, GROUPS = 256 / LANES;
  __shared__ float4 s_o[GROUPS][LANES];
  __shared__ float s_m[GROUPS], s_l[GROUPS];
  const int i = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  if (p.a.fill) {
    const int q_end = p.r.B ? p.r.q_start[p.r.B] : 0;
    if (q_end >= 0) {
      const long per = static_cast<long>(p.a.Hq) * HD / 8, n = (p.r.n - static_cast<long>(q_end)) * per;
      uint4* o = reinterpret_cast<uint4*>(p.a.out) + q_end * per;
      for (long x = (static_cast<long>(i) * gridDim.y + r) * blockDim.x + tid; x < n; x += static_cast<long>(gridDim.x) * gridDim.y * blockDim.x) o[x] = make_uint4(0, 0, 0, 0);
    }
  }
  const int* head = p.meta + i * 8 + 4;
  if (head[0] < 0) return;
  const int b = head[0], h = head[1], r0 = head[2];
  const Row row = load_row(p.r, b);
  const int rr = r0 + r;
  if (rr >= row.nq * p.G) return;
  int parts = 1;
  if (head[3] == 0)
    while (i + parts < n_ctas && p.meta[(i + parts) * 8] >= 0) {
      const bool end = p.meta[(i + parts) * 8 + 3] != 0;
      ++parts;
      if (end) break;
    }
  auto part = [&](int k) -> const float* { return p.ws + (static_cast<long>(i + k) * 2 + (k == 0 ? 1 : 0)) * UR * (HD + 2); };
  const int grp = tid / LANES, ln = tid % LANES;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k = grp; k < parts; k += GROUPS) {
    const float* w = part(k);
    const float mk = w[UR * HD + 2 * r], lk = w[UR * HD + 2 * r + 1];
    const float4 x = *reinterpret_cast<const float4*>(w + r * HD + ln * 4);
    const float mn = fmaxf(m, mk), ref = mn == -INFINITY ? 0.f : mn;
    const float fa = exp2_fast(m - ref), fb = exp2_fast(mk - ref);
    o.x = o.x * fa + x.x * fb; o.y = o.y * fa + x.y * fb; o.z = o.z * fa + x.z * fb; o.w = o.w * fa + x.w * fb;
    l = l * fa + lk * fb;
    m = mn;
  }
  s_o[grp][ln] = o;
  if (ln == 0) { s_m[grp] = m; s_l[grp] = l; }
  __syncthreads();
  if (grp != 0) return;
  float mm = -INFINITY;
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) mm = fmaxf(mm, s_m[k]);
  const float ref = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < GROUPS; ++k) {
    const float f = exp2_fast(s_m[k] - ref);
    const float4 x = s_o[k][ln];
    ll += s_l[k] * f;
    o.x += x.x * f; o.y += x.y * f; o.z += x.z * f; o.w += x.w * f;
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  const __nv_bfloat162 a = __floats2bfloat162_rn(o.x * inv, o.y * inv), c = __floats2bfloat162_rn(o.z * inv, o.w * inv);
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out) + ((static_cast<long>(row.q0) + rr / p.G) * p.a.Hq + h * p.G + rr % p.G) * HD + ln * 4;
  *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
}

namespace {

template <bool FP4, int HD, int NT>
int launch(const AttnK& k, int ctas, cudaStream_t st) {
  using GEO = Geo<FP4, HD, NT>;
  // (set on every call: the attribute belongs to the device that is current, and costs no launch)
  if (cudaFuncSetAttribute(paged_attention_kernel<FP4, HD, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, GEO::SMEM) != cudaSuccess) return 4;
  paged_attention_kernel<FP4, HD, NT><<<ctas, GEO::THREADS, GEO::SMEM, st>>>(k);
  paged_attention_join_kernel<HD, GEO::UR><<<dim3(ctas, GEO::UR), 256, 0, st>>>(k, ctas);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

struct Shape { int ctas, ur, piece; };
template <bool FP4, int HD, int NT> Shape shape() { using GEO = Geo<FP4, HD, NT>; return {GEO::CTAS, GEO::UR, GEO::PIECE}; }

template <bool FP4>
bool shape_of(int hd, int nt, Shape* s) {
  if (hd == 64) { *s = nt == 1 ? shape<FP4, 64, 1>() : nt == 2 ? shape<FP4, 64, 2>() : shape<FP4, 64, 4>(); return true; }
  if (hd == 128) { *s = nt == 1 ? shape<FP4, 128, 1>() : shape<FP4, 128, 2>(); return nt <= 2; }
  if (hd == 256) { *s = nt == 1 ? shape<FP4, 256, 1>() : shape<FP4, 256, 2>(); return nt <= 2; }
  return false;
}

template <bool FP4>
int dispatch(const AttnK& k, int hd, const PagedAttnPlan& plan, cudaStream_t st) {
  switch (hd * 8 + plan.nt) {
    case 64 * 8 + 1: return launch<FP4, 64, 1>(k, plan.ctas, st);
    case 64 * 8 + 2: return launch<FP4, 64, 2>(k, plan.ctas, st);
    case 64 * 8 + 4: return launch<FP4, 64, 4>(k, plan.ctas, st);
    case 128 * 8 + 1: return launch<FP4, 128, 1>(k, plan.ctas, st);
    case 128 * 8 + 2: return launch<FP4, 128, 2>(k, plan.ctas, st);
    case 256 * 8 + 1: return launch<FP4, 256, 1>(k, plan.ctas, st);
    case 256 * 8 + 2: return launch<FP4, 256, 2>(k, plan.ctas, st);
  }
  return 1;
}

}  // namespace

// How many query rows a unit has (8, 16 or 32: the smallest that holds a row's average, so that cached entries are read once)
// and how many CTAs run: as many as are resident, fewer where even full tables have fewer pieces.
int paged_attention_plan(const PagedRows& r, const PagedPool& c, int Hq, int sms, PagedAttnPlan* plan) {
  const int G = Hq / r.Hkv;
  const long per_row = r.B ? static_cast<long>(G) * ((r.n + r.B - 1) / r.B) : 0;
  const int most = c.hd == 64 ? 4 : 2;
  int nt = 1;
  while (nt < most && 8 * nt < per_row) nt *= 2;
  Shape s;
  if (!(c.fp4 ? shape_of<true>(c.hd, nt, &s) : shape_of<false>(c.hd, nt, &s))) return 1;
  const long units = (static_cast<long>(r.n) * G / s.ur + r.B) * r.Hkv;
  const long pieces = ((static_cast<long>(r.width) << r.page_shift) / s.piece + 2) * units;
  long ctas = static_cast<long>(sms) * s.ctas;
  if (pieces < ctas) ctas = pieces;
  plan->nt = nt;
  plan->ctas = ctas < 1 ? 1 : static_cast<int>(ctas);
  plan->ws_floats = static_cast<long>(plan->ctas) * 2 * s.ur * (c.hd + 2);
  plan->ws_ints = static_cast<long>(plan->ctas) * 8;
  return 0;
}

int paged_attention(const PagedRows& r, const PagedPool& c, const PagedAttn& a, const PagedAttnPlan& plan, float* ws, int* meta, cudaStream_t st) {
  if (r.n == 0) return 0;
  if (a.Hq % r.Hkv || (static_cast<long>(r.n_pages) * r.Hkv << r.page_shift) > 0x7fffffffL) return 1;
  // rotating cached keys: pairs within the first 64 channels, whole lanes apart
  if (a.cap && a.half != 8 && a.half != 16 && a.half != 32) return 1;
  AttnK k{r, c, a, a.Hq / r.Hkv, ws, meta};
  return c.fp4 ? dispatch<true>(k, c.hd, plan, st) : dispatch<false>(k, c.hd, plan, st);
}

}  // namespace ghb
