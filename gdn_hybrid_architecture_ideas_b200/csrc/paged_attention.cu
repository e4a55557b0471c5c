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
// scale: exact in f16 (2 + 4 significant bits, 2^-10 .. 2688). Queries are rounded to f16 once (at most 2^-11 of the value), after a
// power of two per query row has brought them to about one, probabilities to f16 (2^-11, scaled up: PSHIFT below), keys that are rotated
// here to f16 (2^-11): beside the 2^-3 that 4 bits cost a value, and the output's own 2^-8 in bfloat16, none of it shows (0.0017 of the outputs' norm
// from 64 bits, the plain form 0.0016). bfloat16 cache: queries, probabilities and the keys that are rotated here as the sum of two
// bfloat16 (2^-16), other keys as they are. The sum of the probabilities is taken over the rounded ones. All sums are float32 in
// the accumulators.
//
// Work: the pieces (one tile of positions for each warp) of all (row, KV head, block of query rows) units form one sequence,
// and every CTA takes an equal share of it, so that rows of any lengths load the SMs evenly. Each CTA finds its share by
// a prefix sum over the rows. Warps take the tiles of a piece and keep their own running softmax; they meet in shared memory at
// the end of a unit's part. A unit cut by CTA borders leaves partial results (at most two a CTA), joined by a second kernel in
// the order of the CTAs: no atomics, the same result every time.
//
// Loads go by cp.async into a ring of tiles private to each warp: no block barrier in the loop, and no warp waits for another. The
// part of a tile that lies in one page is contiguous, so with pages of a tile or more the addresses are one base and constants.
// (Bulk copies cost one instruction instead of nine, but about 32 clocks each in the SM's copy engine, which bound
// the loop; one more warp that loads for all the others ties them to the slowest. Both were measured slower.) What no
// row sees gets scales of zero (4 bits), so that its values are zero; in bfloat16 a tile with masked infinities or NaN is summed
// position by position.
//
// Measured: 64 rows of 32k positions, 16 heads over 4 of 64, under a cap of 2048: 4 bits 155 us (604 MB, 0.59 of the copy's rate; 66% of the
// issue slots: the conversion of every entry for each block of 8 query rows bounds it), bfloat16 363 us (0.90). 8 to 256 such rows in 4 bits
// are 24.6 us and 2.02 us a row, without a cap 19.8 and 1.82 (0.79 of the copy's rate): the fixed part is the share, the queries, the first
// tiles, joining warps and CTAs. 12 rows of up to 9k positions of 2 heads of 256 in bfloat16 35 us for 17 us of bytes, one row 11 us.
#include <atomic>

#include "paged.cuh"

namespace ghb {

struct AttnK {                       // by value to the kernels
  PagedRows r; PagedPool c; PagedAttn a;
  int G;
  float* ws; int* meta;
};

// W warps, ST ring stages each, CTAS a SM, MT 16-position tiles a warp takes at once.
template <bool FP4, int HD> struct Cfg;
template <> struct Cfg<true, 64> { static constexpr int W = 8, ST = 2, CTAS = 2, MT = 4; };
template <> struct Cfg<true, 128> { static constexpr int W = 8, ST = 2, CTAS = 2, MT = 2; };
template <> struct Cfg<true, 256> { static constexpr int W = 8, ST = 2, CTAS = 1, MT = 2; };
template <> struct Cfg<false, 64> { static constexpr int W = 8, ST = 3, CTAS = 2, MT = 1; };
template <> struct Cfg<false, 128> { static constexpr int W = 4, ST = 3, CTAS = 2, MT = 1; };
template <> struct Cfg<false, 256> { static constexpr int W = 6, ST = 2, CTAS = 1, MT = 1; };

constexpr int UNIT_ROWS = 8;         // query rows of a unit: the products' columns

template <bool FP4, int HD>
struct Geo : Cfg<FP4, HD> {
  using B = Cfg<FP4, HD>;
  static constexpr int MT = B::MT, ST = B::ST;
  static constexpr int TILE = 16 * MT;
  static constexpr int H = HD / 64;                  // 64-channel slices
  static constexpr int ROW = FP4 ? HD / 2 : HD * 2;  // bytes of a position
  static constexpr int S = HD / 16;                  // scale bytes of a position
  static constexpr int KB = TILE * ROW;              // bytes of a tile's keys (values the same)
  static constexpr int SB = FP4 ? TILE * S : 0;      // bytes of its scales
  static constexpr int STAGE = 2 * KB + 2 * SB;
  static constexpr int UR = UNIT_ROWS;
  static constexpr int PIECE = B::W * TILE;
  static constexpr int RING = B::W * ST * STAGE;
  static constexpr int MERGE = B::W * UR * HD * 4;
  // Partial outputs beside the ring, where both fit twice on an SM: the next unit's first tiles are then on their way while the
  // warps of this one join. Else over it.
  static constexpr bool BESIDE = FP4 && HD == 64;
  static constexpr int DATA = BESIDE ? RING + MERGE : RING > MERGE ? RING : MERGE;
  static constexpr int QCOPIES = FP4 ? 1 : 2;        // bfloat16: high and low part
  static constexpr int QB = UR * HD * 2;             // bytes of one copy of the queries
  static constexpr int smem(bool cap) { return DATA + (cap ? 2 : 1) * QCOPIES * QB; }      // under a cap: queries by the cap and by their positions
  static constexpr int THREADS = B::W * 32;
};

// Probabilities are exp2(score - reference + PSHIFT): the reference trails the running maximum by at most SLACK, so that it moves (and
// the sums are rescaled, and lanes exchange their maxima) only now and then. f16: up to 2^15, and normal down to 2^-21 of the
// reference; what a smaller one loses is at most 2^-32 of the reference's weight.
constexpr float PSHIFT = 7.f, SLACK = 8.f;
// A condition that is rarely true, kept a branch (as predicated instructions its body would cost every tile).
__device__ __forceinline__ int opaque(int x) { asm volatile("" : "+r"(x)); return x; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
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
// the first product of a sum: no addend
template <bool FP4>
__device__ __forceinline__ void mma_first(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (FP4)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
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
__device__ __forceinline__ uint32_t hmul2_low(uint32_t a, uint32_t b) {        // both by b's low half
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), __low2half2(*reinterpret_cast<const __half2*>(&b)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// eight codes (a 32-bit word) -> four f16 pairs
__device__ __forceinline__ void codes_to_f16(uint32_t w, uint32_t* h) {
  asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\tmov.b32 {c0, c1, c2, c3}, %4;\n\tcvt.rn.f16x2.e2m1x2 %0, c0;\n\tcvt.rn.f16x2.e2m1x2 %1, c1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, c2;\n\tcvt.rn.f16x2.e2m1x2 %3, c3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(w));
}
__device__ __forceinline__ void code_to_f16(uint32_t byte, uint32_t& h) {        // the low byte's two codes
  asm("{\n\t.reg .b8 c0, c1, c2, c3;\n\tmov.b32 {c0, c1, c2, c3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, c0;\n\t}" : "=r"(h) : "r"(byte));
}
// two E4M3 scales (bytes 0 and 1) -> an f16 pair
__device__ __forceinline__ uint32_t scales_to_f16(uint32_t two) {
  uint32_t h;
  asm("{\n\t.reg .b16 c, d;\n\tmov.b32 {c, d}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, c;\n\t}" : "=r"(h) : "r"(two));
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
// what rounding a pair to bfloat16 left, as bfloat16 (an infinity has no remainder)
__device__ __forceinline__ uint32_t rest(float2 x, uint32_t rounded) {
  const float2 f = unpack<false>(rounded);
  return pack<false>(isfinite(x.x) ? x.x - f.x : 0.f, isfinite(x.y) ? x.y - f.y : 0.f);
}
// a byte's low half of a, its high half of b
__device__ __forceinline__ uint32_t low_nibbles(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, 0x0f0f0f0f, 0xe4;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// N neighbouring channels (2, 4 or 8) as float32
template <int N> __device__ __forceinline__ void load_channels(const float* p, float* x) {
  if constexpr (N == 2) { const float2 u = *reinterpret_cast<const float2*>(p); x[0] = u.x; x[1] = u.y; }
  else {
#pragma unroll
    for (int i = 0; i < N; i += 4) { const float4 u = *reinterpret_cast<const float4*>(p + i); x[i] = u.x; x[i + 1] = u.y; x[i + 2] = u.z; x[i + 3] = u.w; }
  }
}
template <int N> __device__ __forceinline__ void load_channels(const __nv_bfloat16* p, float* x) {
  uint32_t w[N / 2];
  if constexpr (N == 2) w[0] = *reinterpret_cast<const uint32_t*>(p);
  else if constexpr (N == 4) { const uint2 u = *reinterpret_cast<const uint2*>(p); w[0] = u.x; w[1] = u.y; }
  else { const uint4 u = *reinterpret_cast<const uint4*>(p); w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w; }
#pragma unroll
  for (int i = 0; i < N / 2; ++i) { const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
}

// Row rho (0 .. 7) of an 8-row group of the tiles is position place(rho) of the group. 4 bits: chosen so that both the keys' reads
// (8 bytes of rows rho = 0..3 or 4..7 at once) and the values' (4 bytes of rows 0,2,4,6 or 1,3,5,7) touch four
// 32-byte rows that differ modulo 4, hence all 32 banks. bfloat16 rows are 128 bytes and swizzled by 16-byte chunk instead.
template <bool FP4> __device__ __forceinline__ int place(int rho) {
  return FP4 ? (rho & 4) | (((rho ^ (rho >> 2)) & 1) << 1) | ((rho >> 1) & 1) : rho;
}

// The units of a row: how many for a head, how many pieces each, and what a unit costs. Under a cap, pieces with keys to rotate count
// 3 where the others, which come first, count 2 (548 against 343 instructions for 32 positions of a head of 64 in 4 bits, 804 against 567
// in bfloat16; 64 rows of 8192 positions in 4 bits, all within the cap 77 us, all beyond 54).
template <bool CAP>
struct RowWork {
  static constexpr int FAR = CAP ? 2 : 1, NEAR = CAP ? 3 : 1;
  int units, pieces, base, far;              // far: leading pieces that lie beyond the cap for every new token
  __device__ __forceinline__ long cost() const { return static_cast<long>(far) * FAR + static_cast<long>(pieces - far) * NEAR; }
  __device__ __forceinline__ long cost_at(int piece) const { return piece < far ? static_cast<long>(piece) * FAR : static_cast<long>(far) * FAR + static_cast<long>(piece - far) * NEAR; }
  // the first piece that starts at a cost of c or more
  __device__ __forceinline__ int piece_at(long c) const {
    const long f = static_cast<long>(far) * FAR;
    return static_cast<int>(c <= f ? (c + FAR - 1) / FAR : far + (c - f + NEAR - 1) / NEAR);
  }
};
template <typename GEO, bool CAP>
__device__ __forceinline__ RowWork<CAP> row_work(const Row& row, int G, int cap) {
  RowWork<CAP> w;
  w.units = (row.nq * G + GEO::UR - 1) / GEO::UR;
  w.base = row.start & ~(GEO::TILE - 1);
  const int span = row.len - w.base;
  w.pieces = span > 0 ? (span + GEO::PIECE - 1) / GEO::PIECE : 1;      // a row that sees nothing still owes zeros
  w.far = 0;
  if (CAP) {
    const int beyond = row.len - row.nq - cap - w.base;                // positions beyond the cap of the first new token
    w.far = beyond > 0 ? min(beyond / GEO::PIECE, w.pieces) : 0;
  }
  return w;
}

// a / b for a >= 0, b > 0: costs fit 32 bits but for enormous batches
__device__ __forceinline__ long quot(long a, long b) {
  return ((a | b) >> 32) == 0 ? static_cast<long>(static_cast<unsigned>(a) / static_cast<unsigned>(b)) : a / b;
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

// STEPS: 0 without a cap, else half / 8: the groups of 8 rotary pairs of the keys that are rotated here (1, 2 or 4).
template <bool FP4, int HD, int STEPS>
__global__ void __launch_bounds__(Geo<FP4, HD>::THREADS, Geo<FP4, HD>::CTAS) paged_attention_kernel(const __grid_constant__ AttnK p) {
  using GEO = Geo<FP4, HD>;
  constexpr bool CAP = STEPS > 0;
  constexpr int H = GEO::H, MT = GEO::MT, TILE = GEO::TILE, UR = GEO::UR, W = GEO::W, ST = GEO::ST;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long s_warp[W];
  __shared__ long s_at[2];
  __shared__ Row s_row;
  __shared__ float s_mul[UR];                 // a query row's factor on its scores: scale * log2(e) * its power of two
  __shared__ float s_m[W][UR], s_l[W][UR];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const PagedRows& R = p.r;
  const int n_ctas = gridDim.x, cta = blockIdx.x, Hkv = R.Hkv, G = p.G;

  // ---- this CTA's share of the pieces
  Row own = {0, 0, 0, 0};
  auto pieces_of = [&](int i) -> long {
    if (i >= R.B) return 0;
    own = load_row(R, i);
    const RowWork<CAP> w = row_work<GEO, CAP>(own, G, p.a.cap);
    return w.units * w.cost() * Hkv;
  };
  long total = 0, mine = 0, ex = 0;
  for (int b0 = 0; b0 < R.B; b0 += GEO::THREADS) {
    long all;
    mine = pieces_of(b0 + tid);
    ex = total + block_scan<GEO::THREADS>(mine, s_warp, &all);
    total += all;
  }
  // CTAs with work: their shares are at least a piece's cost, so that each holds the start of one. The first `extra` have one more.
  const long most = quot(total, RowWork<CAP>::NEAR);
  const long use = most < 1 ? (total > 0) : most < n_ctas ? most : n_ctas;
  int* meta = p.meta + cta * 8;
  if (tid == 0) meta[0] = 0;                  // parts of the unit that this CTA begins and others end
  if (cta >= use) return;
  const long share = quot(total, use), extra = total - share * use;
  auto start_of = [&](long i) -> long { return share * i + (i < extra ? i : extra); };
  auto cta_of = [&](long c) -> long { return c < (share + 1) * extra ? quot(c, share + 1) : extra + quot(c - (share + 1) * extra, share); };
  const long lo = start_of(cta), hi = start_of(cta + 1);
  if (R.B <= GEO::THREADS) {
    if (lo >= ex && lo < ex + mine) { s_at[0] = tid; s_at[1] = ex; s_row = own; }
  } else {
    long before = 0;
    for (int b0 = 0; before <= lo; b0 += GEO::THREADS) {
      long all;
      mine = pieces_of(b0 + tid);
      ex = before + block_scan<GEO::THREADS>(mine, s_warp, &all);
      if (lo >= ex && lo < ex + mine) { s_at[0] = b0 + tid; s_at[1] = ex; s_row = own; }
      before += all;
    }
  }
  __syncthreads();
  int b = static_cast<int>(s_at[0]);
  long row_at = s_at[1];
  Row row = s_row;

  uint8_t* ring = smem + warp * (ST * GEO::STAGE);
  const uint32_t ring_u = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  uint8_t* sq = smem + GEO::DATA;
  const int half = CAP ? 8 * STEPS : p.a.half;
  // ---- the part of a unit that this CTA does next
  struct Part { int b, q0, start, h, r0, n_rows, p0, n_pieces, pieces, pos0, p_first, p_last, tile0; long last_cost; };
  long at = lo;
  Part sg;
  // (at: where the part starts, in costs; its pieces are those that start in at .. hi. Moves at to the part's end; false: none left.)
  auto locate = [&]() -> bool {
    while (at < hi) {
      const RowWork<CAP> wk = row_work<GEO, CAP>(row, G, p.a.cap);
      const long each = wk.cost(), count = wk.units * each * Hkv;
      if (at >= row_at + count) {             // (rows without tokens have no pieces)
        row_at += count;
        row = load_row(R, ++b);
        continue;
      }
      const int unit = static_cast<int>(quot(at - row_at, each));
      const long unit_at = row_at + unit * each;
      sg.p0 = wk.piece_at(at - unit_at);
      const int p1 = hi - unit_at >= each ? wk.pieces : wk.piece_at(hi - unit_at);
      at = min(hi, unit_at + each);
      if (p1 <= sg.p0) continue;
      sg.b = b; sg.q0 = row.q0; sg.start = row.start; sg.pieces = wk.pieces;
      sg.n_pieces = p1 - sg.p0;
      sg.last_cost = unit_at + wk.cost_at(wk.pieces - 1);
      sg.h = unit / wk.units; sg.r0 = (unit % wk.units) * UR;
      sg.n_rows = min(UR, row.nq * G - sg.r0);
      sg.pos0 = row.len - row.nq;                            // position of the row's first new token
      sg.p_first = sg.pos0 + sg.r0 / G;
      sg.p_last = row.len ? sg.pos0 + (sg.r0 + sg.n_rows - 1) / G : -1;
      sg.tile0 = wk.base + sg.p0 * GEO::PIECE + warp * TILE;
      return true;
    }
    return false;
  };
  // ---- loads of one tile: positions tile0 + k PIECE .. + TILE. A tile is one or more chunks, each within a page and so contiguous
  // per head; all lanes copy 16 bytes at a time. Page ids are looked up for 32 chunks at once (32 tiles where a page holds a
  // tile): lane i holds the entry of chunk i of them.
  const int c_shift = min(R.page_shift, TILE == 64 ? 6 : TILE == 32 ? 5 : 4);
  const unsigned all_on = (1u << (TILE >> c_shift)) - 1u;
  const int n_log = TILE == 64 ? 6 - c_shift : TILE == 32 ? 5 - c_shift : 4 - c_shift;          // log2 of a tile's chunks
  int entry = 0;
  unsigned batch_on = 0;
  auto look_up = [&](int k) {                // tiles k .. of this warp
    const int tok = sg.tile0 + (k + (lane >> n_log)) * GEO::PIECE + ((lane & ((1 << n_log) - 1)) << c_shift);
    entry = -1;
    if (k + (lane >> n_log) < sg.n_pieces && tok + (1 << c_shift) > sg.start && tok <= sg.p_last) {
      const int pg = R.pages[sg.b * R.pages_stride + (tok >> R.page_shift)];
      if (pg < 0 || pg >= R.n_pages) *R.err = ST_PAGE;
      else entry = ((pg * Hkv + sg.h) << R.page_shift) + (tok & ((1 << R.page_shift) - 1));
    }
    batch_on = __ballot_sync(0xffffffffu, entry >= 0);
  };
  const uint8_t* k_lane = static_cast<const uint8_t*>(p.c.k) + lane * 16;
  const uint8_t* v_lane = static_cast<const uint8_t*>(p.c.v) + lane * 16;
  constexpr int L = FP4 ? TILE * GEO::S / 16 : 1;          // 16-byte parts of a tile's key scales; its value scales follow
  const uint8_t* s_lane = lane % (2 * L) < L ? p.c.k_scale : p.c.v_scale;
  auto issue = [&](int k, int stage) -> unsigned {         // returns the mask of tile k's chunks that are read
    if ((k & ((32 >> n_log) - 1)) == 0 && k < sg.n_pieces) look_up(k);
    const int at_chunk = (k << n_log) & 31;
    const unsigned on = k < sg.n_pieces ? (batch_on >> at_chunk) & all_on : 0u;
    if (on) {
      const uint32_t st = ring_u + stage * GEO::STAGE;
      constexpr int CH = GEO::ROW / 16, N = TILE * CH / 32;        // 16-byte parts of a position; copies a lane makes of keys
      auto place_of = [&](int pos, int sub) -> uint32_t {          // bfloat16: slices of 128-byte rows, swizzled
        if constexpr (FP4) return pos * GEO::ROW + sub * 16;
        else return (sub >> 3) * (TILE * 128) + pos * 128 + (((sub & 7) ^ (pos & 7)) << 4);
      };
      if (n_log == 0) {                      // the whole tile lies in one page: one address, fixed distances
        const int e = __shfl_sync(0xffffffffu, entry, at_chunk);
        const long off = static_cast<long>(e) * GEO::ROW;
#pragma unroll
        for (int i = 0; i < N; ++i) cp16(st + place_of((i * 32 + lane) / CH, (i * 32 + lane) % CH), k_lane + off + i * 512);
#pragma unroll
        for (int i = 0; i < N; ++i) cp16(st + GEO::KB + place_of((i * 32 + lane) / CH, (i * 32 + lane) % CH), v_lane + off + i * 512);
        if constexpr (FP4) {
          const long soff = static_cast<long>(e) * GEO::S + (lane % L) * 16;
          if constexpr (2 * L > 32) {        // (wide heads: one copy for the keys', one for the values')
            cp16(st + 2 * GEO::KB + lane * 16, p.c.k_scale + soff);
            cp16(st + 2 * GEO::KB + GEO::SB + lane * 16, p.c.v_scale + soff);
          } else if (2 * L == 32 || lane < 2 * L) {
            cp16(st + 2 * GEO::KB + lane * 16, s_lane + soff);
          }
        }
      } else {
        auto copy = [&](uint32_t to, const void* from) {
#pragma unroll
          for (int i = 0; i < N; ++i) {
            const int pos = (i * 32 + lane) / CH, sub = (i * 32 + lane) % CH, c = pos >> c_shift;
            const int e = __shfl_sync(0xffffffffu, entry, at_chunk + c) + (pos & ((1 << c_shift) - 1));
            const bool ok = (on >> c) & 1;
            cp16(to + place_of(pos, sub), static_cast<const uint8_t*>(from) + (ok ? static_cast<long>(e) * GEO::ROW + sub * 16 : 0), ok);
          }
        };
        copy(st, p.c.k);
        copy(st + GEO::KB, p.c.v);
        if constexpr (FP4) {
#pragma unroll
          for (int i = 0; i < (2 * L + 31) / 32; ++i) {
            const int idx = i * 32 + lane, pos = (idx % L) * (16 / GEO::S), c = pos >> c_shift;
            const int e = __shfl_sync(0xffffffffu, entry, at_chunk + c) + (pos & ((1 << c_shift) - 1));
            const bool ok = (on >> c) & 1;
            const uint8_t* base = idx % (2 * L) < L ? p.c.k_scale : p.c.v_scale;
            if (2 * L >= 32 || idx < 2 * L) cp16(st + 2 * GEO::KB + idx * 16, base + (ok ? static_cast<long>(e) * GEO::S : 0), ok);
          }
        }
      }
    }
    cp_commit();
    return on;
  };
  unsigned on_ring[ST];
  auto begin = [&]() {
#pragma unroll
    for (int k = 0; k < ST - 1; ++k) on_ring[k] = issue(k, k);
  };
  if (!locate()) return;
  bool begun = false;
  while (true) {
    const int h = sg.h, r0 = sg.r0, n_rows = sg.n_rows, n_pieces = sg.n_pieces, pos0 = sg.pos0, p_first = sg.p_first, p_last = sg.p_last, tile0 = sg.tile0;
    const int q0 = sg.q0, start = sg.start, p0 = sg.p0, pieces = sg.pieces;
    int stage = 0;                             // of tile k

    // ---- the unit's queries, a warp a row: all loads first (they and the first tiles are under way together), then rotated (by their
    // positions; under a cap one copy by the cap and one by the positions), brought to about one, in the products' order
    // (a lane takes HD / 32 neighbouring channels: 2, 4 or 8, which divides half, so that their partners are neighbours too)
    constexpr int RPW = (UR + W - 1) / W, CPL = HD / 32;
    const int c0 = lane * CPL;
    const bool turns = c0 < 2 * half, low = c0 < half;
    constexpr int TURNS = CAP ? 2 : 1;         // the copies' rotations: of the plain products, of the rotating ones
    float x[RPW][CPL], y[RPW][CPL], co[TURNS][RPW][CPL], si[TURNS][RPW][CPL];
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
      const int r = warp + j * W, rr = r0 + r;
      const bool live = r < n_rows && p_last >= 0;
      // (addresses are clamped to valid ones instead of branched over, so that the loads stand side by side)
      const int i = live ? rr / G : 0, head = h * G + (live ? rr % G : 0);
      const long off = (static_cast<long>(q0) + i) * p.a.q_ts + head * p.a.q_hs;
      int at_pos = pos0 + i - start;
      if (live && half > 0 && at_pos >= p.a.n_pos) { *R.err = ST_ROPE; at_pos = p.a.n_pos - 1; }
      const int partner = turns ? (low ? c0 + half : c0 - half) : c0;
      if (p.a.q_f32) {
        load_channels<CPL>(static_cast<const float*>(p.a.q) + off + c0, x[j]);
        load_channels<CPL>(static_cast<const float*>(p.a.q) + off + partner, y[j]);
      } else {
        load_channels<CPL>(static_cast<const __nv_bfloat16*>(p.a.q) + off + c0, x[j]);
        load_channels<CPL>(static_cast<const __nv_bfloat16*>(p.a.q) + off + partner, y[j]);
      }
      if (half > 0) {
#pragma unroll
        for (int w = 0; w < TURNS; ++w) {
          const long e = static_cast<long>(CAP && w == 0 ? p.a.cap : max(0, min(at_pos, p.a.n_pos - 1))) * half + (turns ? (low ? c0 : c0 - half) : 0);
          load_channels<CPL>(p.a.cos + e, co[w][j]);
          load_channels<CPL>(p.a.sin + e, si[w][j]);
        }
      }
    }
    if (!begun) begin();
    begun = true;
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
      const int r = warp + j * W;
      if (r >= UR) break;
      const bool live = r < n_rows && p_last >= 0;
      float top = 0.f;
#pragma unroll
      for (int i = 0; i < CPL; ++i) { x[j][i] = live ? x[j][i] : 0.f; y[j][i] = live ? y[j][i] : 0.f; }
#pragma unroll
      for (int i = 0; i < CPL; ++i) top = fmaxf(top, fabsf(x[j][i]));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      int ex = 0;
      if (FP4 && top > 0.f && top < INFINITY) ex = ilogbf(top);
      ex = max(-120, min(120, ex));
      const float down = exp2f(static_cast<float>(-ex));
      if (lane == 0) s_mul[r] = p.a.scale * 1.44269504088896340736f * exp2f(static_cast<float>(ex));
      float turned[TURNS][CPL];
#pragma unroll
      for (int i = 0; i < CPL; ++i)
#pragma unroll
        for (int w = 0; w < TURNS; ++w) turned[w][i] = (turns ? x[j][i] * co[w][j][i] + y[j][i] * (low ? -si[w][j][i] : si[w][j][i]) : x[j][i]) * down;
      // Two channels at a time to their places: in the order of the plain products (a lane owns the 16 channels 16 t .. of each slice),
      // and of the rotating ones (its channels are 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of every block of 16).
      auto put = [&](uint8_t* to, int idx, float a, float z) {
        const uint32_t hi = pack<FP4>(a, z);
        *reinterpret_cast<uint32_t*>(to + idx * 2) = hi;
        if constexpr (!FP4) *reinterpret_cast<uint32_t*>(to + GEO::QB + idx * 2) = rest(make_float2(a, z), hi);
      };
#pragma unroll
      for (int i = 0; i < CPL; i += 2) {
        const int c = c0 + i, cc = c & 63;
        put(sq, ((((c >> 6) * 4 + ((cc & 15) >> 2)) * 32 + r * 4 + (cc >> 4)) << 2) + (cc & 3), turned[0][i], turned[0][i + 1]);
        if constexpr (CAP) put(sq + GEO::QCOPIES * GEO::QB, (((c >> 4) * 32 + r * 4 + ((c & 7) >> 1)) << 2) + ((c >> 2) & 2), turned[1][i], turned[1][i + 1]);
      }
    }
    __syncthreads();

    float mul[2], m[2], l[4];       // l: the sums of the probabilities, as a product with ones (every row the same)
    int prow[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * t + e;
      mul[e] = s_mul[r];
      prow[e] = r < n_rows && p_last >= 0 ? pos0 + (r0 + r) / G : -1;
      m[e] = -INFINITY; l[e] = l[e + 2] = 0.f;
    }
    float o[H * 4][4];
#pragma unroll
    for (int i = 0; i < H * 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

    for (int k = 0; k < n_pieces; ++k) {
      const int first = tile0 + k * GEO::PIECE;
      on_ring[ST - 1] = issue(k + ST - 1, stage == 0 ? ST - 1 : stage - 1);
      const unsigned on = on_ring[0];
#pragma unroll
      for (int i = 0; i < ST - 1; ++i) on_ring[i] = on_ring[i + 1];        // the masks travel with the ring
      uint8_t* st = ring + stage * GEO::STAGE;
      cp_wait<ST - 1>();
      __syncwarp();
      stage = stage == ST - 1 ? 0 : stage + 1;
      if (on) {
        const bool masked = on != all_on || first < start || first + TILE - 1 > p_first;
        if (FP4 && masked) {
          // What no row sees may hold anything: its scales become zero, so that its values are zero. A scale that is not a number
          // where some rows see it and others do not: zero too, and the block's channels of the rows that see it are set by hand.
          bool odd = false;
          for (int pos = lane; pos < TILE; pos += 32) {
            uint32_t* sw = reinterpret_cast<uint32_t*>(st + 2 * GEO::KB + GEO::SB + pos * GEO::S);
            const bool hidden = !((on >> (pos >> c_shift)) & 1) || first + pos < start || first + pos > p_last;
#pragma unroll
            for (int i = 0; i < GEO::S / 4; ++i) {
              if (hidden) sw[i] = 0u;
              odd |= (((sw[i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0u;
            }
          }
          __syncwarp();
#pragma unroll 1
          for (int again = opaque(__any_sync(0xffffffffu, odd)); again > 0; again = opaque(0)) {
#pragma unroll 1
            for (int pos = 0; pos < TILE; ++pos)
#pragma unroll
              for (int hs = 0; hs < H; ++hs) {
                uint8_t* sb = st + 2 * GEO::KB + GEO::SB + pos * GEO::S + hs * 4 + (g >> 1);
                const bool nan = (*sb & 0x7f) == 0x7f;
                __syncwarp();
                if (nan) {
                  *sb = 0;
#pragma unroll
                  for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (first + pos <= prow[e & 1]) o[hs * 4 + i][e] = NAN;
                }
              }
            __syncwarp();
          }
        }
        float s[MT][4];
        // Products that add into one accumulator wait for one another: wide heads take two by turns of their slices, bfloat16 two more
        // for the low parts, summed at the end (a head of 256 is 32 products otherwise in one chain).
        constexpr int CHAINS = (H > 1 ? 2 : 1) * GEO::QCOPIES;
        // one k16 step of the 16 positions of tile mt against the queries' operand at qs (the low parts' `low` bytes further)
        auto step = [&](float (&acc)[CHAINS][4], const uint32_t* a, const uint8_t* qs, int low, int hs, bool begin) {
          const int c = (H > 1 ? hs & 1 : 0) * GEO::QCOPIES;
          const uint2 q1 = *reinterpret_cast<const uint2*>(qs + lane * 8);
          if (begin) mma_first<FP4>(acc[c], a, q1.x, q1.y);
          else mma<FP4>(acc[c], a, q1.x, q1.y);
          if constexpr (!FP4) {
            const uint2 q2 = *reinterpret_cast<const uint2*>(qs + low + lane * 8);
            if (begin) mma_first<FP4>(acc[c + 1], a, q2.x, q2.y);
            else mma<FP4>(acc[c + 1], a, q2.x, q2.y);
          }
        };
        auto joined = [&](float (&acc)[CHAINS][4], int e) -> float {
          float x = acc[0][e];
#pragma unroll
          for (int c = 1; c < CHAINS; ++c) x += acc[c][e];
          return x;
        };
        const bool far_any = !CAP || p_last - first > p.a.cap;                     // some (row, position) beyond the cap
        const bool near_any = CAP && p_first - (first + TILE - 1) <= p.a.cap;      // some within it
        if (far_any) {
          // ---- keys as cached: a lane owns 16 consecutive channels of a slice (4 bits: one block)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float acc[CHAINS][4];
#pragma unroll
            for (int hs = 0; hs < H; ++hs) {
              uint32_t x[2][8];                // [row g or g + 8][channel pair]: channels 16 t + 2 i of slice hs
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int pos = mt * 16 + e * 8 + place<FP4>(g);
                if constexpr (FP4) {
                  const uint2 w = *reinterpret_cast<const uint2*>(st + pos * GEO::ROW + hs * 32 + t * 8);
                  const uint32_t sc = scales_to_f16(st[2 * GEO::KB + pos * GEO::S + hs * 4 + t]);
                  codes_to_f16(w.x, x[e]);
                  codes_to_f16(w.y, x[e] + 4);
#pragma unroll
                  for (int i = 0; i < 8; ++i) x[e][i] = hmul2_low(x[e][i], sc);
                } else {
#pragma unroll
                  for (int c = 0; c < 2; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4*>(st + hs * (TILE * 128) + pos * 128 + (((2 * t + c) ^ (pos & 7)) << 4));
                    x[e][4 * c] = w.x; x[e][4 * c + 1] = w.y; x[e][4 * c + 2] = w.z; x[e][4 * c + 3] = w.w;
                  }
                }
              }
#pragma unroll
              for (int ks = 0; ks < 4; ++ks) {
                const uint32_t a[4] = {x[0][2 * ks], x[1][2 * ks], x[0][2 * ks + 1], x[1][2 * ks + 1]};
                step(acc, a, sq + (hs * 4 + ks) * 256, GEO::QB, hs, hs < 2 && ks == 0);
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][e] = joined(acc, e);
          }
        }
        if constexpr (CAP) {
          if (near_any) {
            // ---- keys within the cap, R(p) q . R(t) k: the keys are rotated here by the table's rows of their positions (any rows: nothing
            // is assumed of how they follow one another). A lane owns channels 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of every block of 16, so
            // that both channels of a rotary pair (half 8, 16 or 32 apart) are its own. A key's row is read by the four lanes that hold its
            // channels, 32 bytes at a time, for the next 16 positions while these are scored.
            float2 co[2][STEPS], si[2][STEPS], co_next[2][STEPS], si_next[2][STEPS];
            auto load_rows = [&](int mt) {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const int d = max(0, min(first + mt * 16 + e * 8 + place<FP4>(g) - start, p.a.n_pos - 1));
                const long at = static_cast<long>(d) * half + 2 * t;
#pragma unroll
                for (int i = 0; i < STEPS; ++i) {
                  co_next[e][i] = __ldg(reinterpret_cast<const float2*>(p.a.cos + at + 8 * i));
                  si_next[e][i] = __ldg(reinterpret_cast<const float2*>(p.a.sin + at + 8 * i));
                }
              }
            };
            load_rows(0);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              float acc[CHAINS][4];
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int i = 0; i < STEPS; ++i) { co[e][i] = co_next[e][i]; si[e][i] = si_next[e][i]; }
              if (mt + 1 < MT) load_rows(mt + 1);
#pragma unroll
              for (int hs = 0; hs < H; ++hs) {
                uint32_t x[2][4][2];           // [row][block of the slice][channels 2 t.. or 2 t + 8 ..]
                uint32_t low[2][4][2];         // bfloat16: what rounding the rotated channels left (the blocks below STEPS)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                  const int pos = mt * 16 + e * 8 + place<FP4>(g);
                  if constexpr (FP4) {
                    const uint32_t scw = *reinterpret_cast<const uint32_t*>(st + 2 * GEO::KB + pos * GEO::S + hs * 4);
                    const uint32_t sc[2] = {scales_to_f16(scw & 0xffffu), scales_to_f16(scw >> 16)};
#pragma unroll
                    for (int bl = 0; bl < 4; ++bl) {
                      const uint2 w = *reinterpret_cast<const uint2*>(st + pos * GEO::ROW + hs * 32 + bl * 8);
                      const uint32_t two = prmt(w.x, w.y, t | ((t + 4) << 4));
                      const uint32_t sb = prmt(sc[bl >> 1], 0u, bl & 1 ? 0x3232 : 0x1010);
                      code_to_f16(two, x[e][bl][0]);
                      code_to_f16(two >> 8, x[e][bl][1]);
                      x[e][bl][0] = hmul2(x[e][bl][0], sb);
                      x[e][bl][1] = hmul2(x[e][bl][1], sb);
                    }
                  } else {
#pragma unroll
                    for (int bl = 0; bl < 4; ++bl)
#pragma unroll
                      for (int c = 0; c < 2; ++c)
                        x[e][bl][c] = *reinterpret_cast<const uint32_t*>(st + hs * (TILE * 128) + pos * 128 + (((2 * bl + c) ^ (pos & 7)) << 4) + t * 4);
                  }
                  if (hs == 0) {
                    // group i of 8 pairs: channels 8 i + 2 t .. with those `half` further
#pragma unroll
                    for (int i = 0; i < STEPS; ++i) {
                      uint32_t &a = x[e][i >> 1][i & 1], &bb = x[e][(i + STEPS) >> 1][(i + STEPS) & 1];
                      const float2 u = unpack<FP4>(a), v = unpack<FP4>(bb), c = co[e][i], n = si[e][i];
                      const float2 ra = make_float2(u.x * c.x - v.x * n.x, u.y * c.y - v.y * n.y), rb = make_float2(v.x * c.x + u.x * n.x, v.y * c.y + u.y * n.y);
                      a = pack<FP4>(ra.x, ra.y);
                      bb = pack<FP4>(rb.x, rb.y);
                      if constexpr (!FP4) { low[e][i >> 1][i & 1] = rest(ra, a); low[e][(i + STEPS) >> 1][(i + STEPS) & 1] = rest(rb, bb); }
                    }
                  }
                }
#pragma unroll
                for (int bl = 0; bl < 4; ++bl) {
                  const uint32_t a[4] = {x[0][bl][0], x[1][bl][0], x[0][bl][1], x[1][bl][1]};
                  const uint8_t* qs = sq + GEO::QCOPIES * GEO::QB + (hs * 4 + bl) * 256;
                  step(acc, a, qs, GEO::QB, hs, hs < 2 && bl == 0);
                  if constexpr (!FP4) {
                    if (hs == 0 && bl < STEPS) {
                      const uint32_t a2[4] = {low[0][bl][0], low[1][bl][0], low[0][bl][1], low[1][bl][1]};
                      const uint2 q1 = *reinterpret_cast<const uint2*>(qs + lane * 8);
                      mma<FP4>(acc[1], a2, q1.x, q1.y);
                    }
                  }
                }
              }
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int tok = first + mt * 16 + (e >> 1) * 8 + place<FP4>(g);
                if (!far_any || prow[e & 1] - tok <= p.a.cap) s[mt][e] = joined(acc, e);
              }
            }
          }
        }
        // ---- masks, where any (row, position) of the tile is not visible
#pragma unroll 1
        for (int again = opaque(masked); again > 0; again = opaque(0)) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int pos = mt * 16 + (e >> 1) * 8 + place<FP4>(g);
              if (!((on >> (pos >> c_shift)) & 1) || first + pos < start || first + pos > prow[e & 1]) s[mt][e] = -INFINITY;
            }
        }
        // ---- the reference of the exponents, where a score leaves the slack (raw scores: the factor is positive)
        float mx[2];
        bool grew = false;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float x = fmaxf(s[0][e], s[0][e + 2]);
#pragma unroll
          for (int mt = 1; mt < MT; ++mt) x = fmaxf(x, fmaxf(s[mt][e], s[mt][e + 2]));
          mx[e] = x * mul[e];
          grew |= mx[e] > m[e] + SLACK;
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float x = mx[e];
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float mn = fmaxf(m[e], x);
            const float alpha = mn == -INFINITY ? 1.f : exp2_fast(m[e] - mn);
            m[e] = mn;
            l[e] *= alpha; l[e + 2] *= alpha;
#pragma unroll
            for (int i = 0; i < H * 4; ++i) { o[i][e] *= alpha; o[i][e + 2] *= alpha; }
          }
        }
        // ---- probabilities
        constexpr int PARTS = FP4 ? 1 : 2;         // bfloat16: what the rounding leaves as a second part (2^-16 together)
        uint32_t pk[PARTS][MT][2];
        const float ref0 = (m[0] == -INFINITY ? 0.f : -m[0]) + (FP4 ? PSHIFT : 0.f), ref1 = (m[1] == -INFINITY ? 0.f : -m[1]) + (FP4 ? PSHIFT : 0.f);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float a = exp2_fast(fmaf(s[mt][2 * q], mul[0], ref0)), z = exp2_fast(fmaf(s[mt][2 * q + 1], mul[1], ref1));
            pk[0][mt][q] = pack<FP4>(a, z);
            if constexpr (PARTS > 1) { const float2 f = unpack<FP4>(pk[0][mt][q]); pk[1][mt][q] = pack<FP4>(a - f.x, z - f.y); }
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
              if (!((on >> (j >> c_shift)) & 1) || first + j < start) continue;
              const float2 p1 = unpack<FP4>(__shfl_sync(0xffffffffu, j < 8 ? pk[0][0][0] : pk[0][0][1], (j & 7) * 4 + t));
              const float2 p2 = unpack<FP4>(__shfl_sync(0xffffffffu, j < 8 ? pk[1][0][0] : pk[1][0][1], (j & 7) * 4 + t));
              const float2 pp = make_float2(p1.x + p2.x, p1.y + p2.y);
              const bool see0 = first + j <= prow[0], see1 = first + j <= prow[1];
              if (see0) { l[0] += pp.x; l[2] += pp.x; }
              if (see1) { l[1] += pp.y; l[3] += pp.y; }
#pragma unroll
              for (int hs = 0; hs < H; ++hs) {
                const uint4 w = *reinterpret_cast<const uint4*>(st + GEO::KB + hs * (TILE * 128) + j * 128 + ((g ^ (j & 7)) << 4));
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float2 v = unpack<FP4>(ws[i]);
                  float* oo = o[hs * 4 + i];
                  if (see0) { oo[0] += pp.x * v.x; oo[2] += pp.x * v.y; }
                  if (see1) { oo[1] += pp.y * v.x; oo[3] += pp.y * v.y; }
                }
              }
            }
          }
        }
        if (plain) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t pb[PARTS][2];
#pragma unroll
            for (int w = 0; w < PARTS; ++w) { pb[w][0] = transpose8(pk[w][mt][0]); pb[w][1] = transpose8(pk[w][mt][1]); }
            constexpr uint32_t ONE2 = FP4 ? 0x3c003c00u : 0x3f803f80u;
            const uint32_t ones[4] = {ONE2, ONE2, ONE2, ONE2};
#pragma unroll
            for (int w = 0; w < PARTS; ++w) mma<FP4>(l, ones, pb[w][0], pb[w][1]);
            const int u0 = mt * 16 + place<FP4>(2 * t), u1 = mt * 16 + place<FP4>(2 * t + 1);
#pragma unroll
            for (int hs = 0; hs < H; ++hs) {
              uint32_t a4[4][4];                   // [channel 8 g + 2 i of the slice][operand register]
              uint32_t sc[2];
              bool second = PARTS > 1;
              if constexpr (FP4) {
                // the codes of positions u0, u1 side by side in a byte, even channels and odd ones: one conversion gives the pair
                const uint8_t* vb = st + GEO::KB + hs * 32 + g * 4;
                const uint32_t w0 = *reinterpret_cast<const uint32_t*>(vb + u0 * GEO::ROW), w1 = *reinterpret_cast<const uint32_t*>(vb + u1 * GEO::ROW);
                const uint32_t w2 = *reinterpret_cast<const uint32_t*>(vb + (u0 + 8) * GEO::ROW), w3 = *reinterpret_cast<const uint32_t*>(vb + (u1 + 8) * GEO::ROW);
                uint32_t c0[4], c1[4], c2[4], c3[4];
                codes_to_f16(low_nibbles(w0, w1 << 4), c0);
                codes_to_f16(low_nibbles(w0 >> 4, w1), c1);
                codes_to_f16(low_nibbles(w2, w3 << 4), c2);
                codes_to_f16(low_nibbles(w2 >> 4, w3), c3);
                const uint8_t* sb = st + 2 * GEO::KB + GEO::SB + hs * 4;
                auto scale_of = [&](int u) { return *reinterpret_cast<const uint32_t*>(sb + u * GEO::S); };
                const uint32_t pick = (g >> 1) | ((4 + (g >> 1)) << 4);            // this lane's block of both
                sc[0] = scales_to_f16(prmt(scale_of(u0), scale_of(u1), pick));
                sc[1] = scales_to_f16(prmt(scale_of(u0 + 8), scale_of(u1 + 8), pick));
#pragma unroll
                for (int i = 0; i < 4; ++i) { a4[i][0] = hmul2(c0[i], sc[0]); a4[i][1] = hmul2(c1[i], sc[0]); a4[i][2] = hmul2(c2[i], sc[1]); a4[i][3] = hmul2(c3[i], sc[1]); }
              } else {
                const uint8_t* vb = st + GEO::KB + hs * (TILE * 128);
                uint32_t v[4][4];                  // [position u0, u1, u0 + 8, u1 + 8][channel pair 8 g + 2 i]
                const int us[4] = {u0, u1, u0 + 8, u1 + 8};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                  const uint4 w = *reinterpret_cast<const uint4*>(vb + us[c] * 128 + ((g ^ (us[c] & 7)) << 4));
                  v[c][0] = w.x; v[c][1] = w.y; v[c][2] = w.z; v[c][3] = w.w;
                }
                // An infinite value stays infinite: a weight's second part may be zero or negative, and is left out beside one.
                __nv_bfloat162 zero = __floats2bfloat162_rn(0.f, 0.f), odd = zero;
#pragma unroll
                for (int c = 0; c < 4; ++c)
#pragma unroll
                  for (int i = 0; i < 4; ++i) odd = __hfma2(*reinterpret_cast<const __nv_bfloat162*>(&v[c][i]), zero, odd);      // NaN from there on
                second = !__any_sync(0xffffffffu, (*reinterpret_cast<const uint32_t*>(&odd) & 0x7fff7fffu) != 0u);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  a4[i][0] = prmt(v[0][i], v[1][i], 0x5410); a4[i][1] = prmt(v[0][i], v[1][i], 0x7632);
                  a4[i][2] = prmt(v[2][i], v[3][i], 0x5410); a4[i][3] = prmt(v[2][i], v[3][i], 0x7632);
                }
              }
#pragma unroll
              for (int i = 0; i < 4; ++i) mma<FP4>(o[hs * 4 + i], a4[i], pb[0][0], pb[0][1]);
              if (second) {
#pragma unroll
                for (int i = 0; i < 4; ++i) mma<FP4>(o[hs * 4 + i], a4[i], pb[PARTS - 1][0], pb[PARTS - 1][1]);
              }
            }
          }
        }
      }
      __syncwarp();          // the stage is consumed before the next issue refills it
    }
    cp_wait<0>();
    if constexpr (!GEO::BESIDE) __syncthreads();         // every warp is done with its ring: the region takes the partial outputs

    // ---- join the warps
    float* so = reinterpret_cast<float*>(smem + (GEO::BESIDE ? GEO::RING : 0));
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 2 * t + e;
      if (g == 0) { s_m[warp][r] = m[e]; s_l[warp][r] = l[e]; }
      float* dst = so + (static_cast<long>(warp) * UR + r) * HD + 8 * g;
#pragma unroll
      for (int i = 0; i < H * 4; ++i)
        *reinterpret_cast<float2*>(dst + (i >> 2) * 64 + (i & 3) * 2) = make_float2(o[i][e], o[i][e + 2]);
    }
    const long last_cost = sg.last_cost;
    const bool more = locate();                // (the next part, from here on)
    if (!more) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (GEO::BESIDE && more) begin();          // (`begun` stays true)
    __syncthreads();
    const bool begins = p0 == 0, ends = p0 + n_pieces == pieces;
    const int slot = begins ? 1 : 0;
    float* wo = p.ws + (static_cast<long>(cta) * 2 + slot) * UR * (HD + 2);
    for (int idx = tid; idx < n_rows * (HD / 4); idx += GEO::THREADS) {
      const int r = idx / (HD / 4), c = idx % (HD / 4) * 4;
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < W; ++w) mm = fmaxf(mm, s_m[w][r]);
      const float ref = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < W; ++w) {            // (a warp that saw nothing holds zeros)
        const float f = exp2_fast(s_m[w][r] - ref);
        const float4 z = *reinterpret_cast<const float4*>(so + (w * UR + r) * HD + c);
        ll += s_l[w][r] * f;
        oo.x += z.x * f; oo.y += z.y * f; oo.z += z.z * f; oo.w += z.w * f;
      }
      if (half > 0 && pos0 + (r0 + r) / G - start >= p.a.n_pos) {        // a query behind the rope table (reported above): left out, zeros
        mm = -INFINITY; ll = 0.f; oo = make_float4(0.f, 0.f, 0.f, 0.f);
      }
      if (begins && ends) {
        const int rr = r0 + r;
        const float inv = ll == 0.f ? 0.f : 1.f / ll;          // a row without a score above -inf has no weights: zeros
        const uint2 out = make_uint2(pack<false>(oo.x * inv, oo.y * inv), pack<false>(oo.z * inv, oo.w * inv));
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.a.out) + ((static_cast<long>(q0) + rr / G) * p.a.Hq + h * G + rr % G) * HD + c) = out;
      } else {
        *reinterpret_cast<float4*>(wo + r * HD + c) = oo;
        if (c == 0) { wo[UR * HD + 2 * r] = mm; wo[UR * HD + 2 * r + 1] = ll; }
      }
    }
    if (tid == 0 && begins && !ends) {           // the first part: how many CTAs hold the others follows from the shares
      meta[1] = h; meta[2] = r0; meta[3] = n_rows; meta[4] = q0;
      meta[0] = static_cast<int>(cta_of(last_cost)) - cta + 1;
    }
    if (!more) break;
    if constexpr (!GEO::BESIDE) {
      __syncthreads();
      begin();
    }
  }
}

// Zeros for the packed tokens that no row owns (those a row owns are written where its units are joined), by all blocks of a launch side
// by side. With q_start in order they lie before q_start[0] and behind q_start[B]. Out of order (status 301), the rows whose own range is
// right keep their tokens, so every token asks all rows.
template <int HD>
__device__ __forceinline__ void zero_unowned(const AttnK& p, int block, int blocks) {
  const PagedRows& R = p.r;
  const long per = static_cast<long>(p.a.Hq) * HD / 8, stride = static_cast<long>(blocks) * blockDim.x, at = static_cast<long>(block) * blockDim.x + threadIdx.x;
  uint4* out = reinterpret_cast<uint4*>(p.a.out);
  bool wrong = false;
  for (int b = threadIdx.x; b <= R.B; b += blockDim.x) { const int q = R.q_start[b]; wrong |= q < 0 || q > R.n || (b < R.B && R.q_start[b + 1] < q); }
  wrong = __syncthreads_or(wrong);
  if (!wrong) {
    const long lead = R.q_start[0] * per, gap = R.q_start[R.B] * per - lead, n = R.n * per - gap;
    for (long x = at; x < n; x += stride) out[x < lead ? x : x + gap] = make_uint4(0, 0, 0, 0);
    return;
  }
  for (long x = at; x < R.n * per; x += stride) {
    const int j = static_cast<int>(x / per);
    bool owned = false;
    for (int b = 0; b < R.B && !owned; ++b) { const int q0 = R.q_start[b], q1 = R.q_start[b + 1]; owned = q0 >= 0 && q1 <= R.n && j >= q0 && j < q1; }
    if (!owned) out[x] = make_uint4(0, 0, 0, 0);
  }
}

// Joins the parts of every unit that CTA borders cut: part one is the last thing its first CTA did (slot 1), the others are the
// first thing that the following CTAs did (slot 0). Block (i, r) joins query row r of the unit whose first part CTA i holds. Also the zeros of
// the packed tokens that no row owns, where the output is this call's own.
template <int HD>
__global__ void __launch_bounds__(256) paged_attention_join_kernel(const __grid_constant__ AttnK p, int n_ctas) {
  constexpr int LANES = HD / 4, GROUPS = 256 / LANES, UR = UNIT_ROWS;
  __shared__ float4 s_o[GROUPS][LANES];
  __shared__ float s_m[GROUPS], s_l[GROUPS];
  const int i = blockIdx.x, r = blockIdx.y, tid = threadIdx.x;
  if (p.a.fill) zero_unowned<HD>(p, i * gridDim.y + r, gridDim.x * gridDim.y);        // (the first kernel writes none of these)
  asm volatile("griddepcontrol.wait;" ::: "memory");          // launched while the first kernel ends; from here on that is complete
  const int* head = p.meta + i * 8;
  const int parts = head[0];
  if (parts == 0 || r >= head[3]) return;
  const int h = head[1], rr = head[2] + r, q0 = head[4];
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
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.a.out) + ((static_cast<long>(q0) + rr / p.G) * p.a.Hq + h * p.G + rr % p.G) * HD + ln * 4;
  *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&c));
}

namespace {

template <bool FP4, int HD, int STEPS>
int launch(const AttnK& k, int ctas, cudaStream_t st) {
  using GEO = Geo<FP4, HD>;
  constexpr int bytes = GEO::smem(STEPS > 0);
  static std::atomic<uint64_t> ready[4];         // devices on which the size is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 4;
  if (dev > 255 || !(ready[dev >> 6].load(std::memory_order_acquire) >> (dev & 63) & 1)) {
    if (cudaFuncSetAttribute(paged_attention_kernel<FP4, HD, STEPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return 4;
    if (dev <= 255) ready[dev >> 6].fetch_or(uint64_t(1) << (dev & 63), std::memory_order_release);
  }
  paged_attention_kernel<FP4, HD, STEPS><<<ctas, GEO::THREADS, bytes, st>>>(k);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, GEO::UR);
  cfg.blockDim = dim3(256);
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, paged_attention_join_kernel<HD>, k, ctas) != cudaSuccess) return 4;
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}
template <bool FP4, int HD>
int launch(const AttnK& k, int ctas, cudaStream_t st) {
  if (!k.a.cap) return launch<FP4, HD, 0>(k, ctas, st);
  return k.a.half == 8 ? launch<FP4, HD, 1>(k, ctas, st) : k.a.half == 16 ? launch<FP4, HD, 2>(k, ctas, st) : launch<FP4, HD, 4>(k, ctas, st);
}

template <bool FP4>
int dispatch(const AttnK& k, int hd, int ctas, cudaStream_t st) {
  switch (hd) {
    case 64: return launch<FP4, 64>(k, ctas, st);
    case 128: return launch<FP4, 128>(k, ctas, st);
    case 256: return launch<FP4, 256>(k, ctas, st);
  }
  return 1;
}

struct Shape { int ctas, piece; };
template <bool FP4, int HD> Shape shape() { using GEO = Geo<FP4, HD>; return {GEO::CTAS, GEO::PIECE}; }
template <bool FP4> Shape shape_of(int hd) { return hd == 64 ? shape<FP4, 64>() : hd == 128 ? shape<FP4, 128>() : shape<FP4, 256>(); }

}  // namespace

// How many CTAs run: as many as are resident, fewer where even full tables have fewer pieces. A unit is always 8 query rows, so that every
// further block of them loads and converts the row's entries again: 24 rows of 16k positions in 4 bits, 32 heads over 8, under a cap
// take 77 us for 1 or 2 new tokens a row, 132 for 4, 179 for 6, 234 for 8. Units of 16 and 24 rows leave room for fewer
// warps and shorter tiles; they were slower than 8 in an earlier form of this loop and are not in the code, so that no figure compares
// them with this one.
int paged_attention_plan(const PagedRows& r, const PagedPool& c, int Hq, int sms, PagedAttnPlan* plan) {
  if (c.hd != 64 && c.hd != 128 && c.hd != 256) return 1;
  const int G = Hq / r.Hkv;
  const Shape s = c.fp4 ? shape_of<true>(c.hd) : shape_of<false>(c.hd);
  const long units = (static_cast<long>(r.n) * G / UNIT_ROWS + r.B) * r.Hkv;
  const long pieces = ((static_cast<long>(r.width) << r.page_shift) / s.piece + 2) * units;
  long ctas = static_cast<long>(sms) * s.ctas;
  if (pieces < ctas) ctas = pieces;
  plan->ctas = ctas < 1 ? 1 : static_cast<int>(ctas);
  plan->ws_floats = static_cast<long>(plan->ctas) * 2 * UNIT_ROWS * (c.hd + 2);
  plan->ws_ints = static_cast<long>(plan->ctas) * 8;
  return 0;
}

int paged_attention(const PagedRows& r, const PagedPool& c, const PagedAttn& a, const PagedAttnPlan& plan, float* ws, int* meta, cudaStream_t st) {
  if (r.n == 0) return 0;
  if (a.Hq % r.Hkv || (static_cast<long>(r.n_pages) * r.Hkv << r.page_shift) > 0x7fffffffL) return 1;
  // rotating cached keys: pairs within the first 64 channels, whole lanes apart
  if (a.cap && a.half != 8 && a.half != 16 && a.half != 32) return 1;
  AttnK k{r, c, a, a.Hq / r.Hkv, ws, meta};
  return c.fp4 ? dispatch<true>(k, c.hd, plan.ctas, st) : dispatch<false>(k, c.hd, plan.ctas, st);
}

}  // namespace ghb
