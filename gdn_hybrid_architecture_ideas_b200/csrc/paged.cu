// Appending to and reading from a paged key/value cache in bfloat16 or 4 bits (layout and checks: paged.cuh).
//
// Append: one thread owns 16 consecutive channels (one 4-bit block) of one token, in one key or value head or in several: loads of 32
// bytes, the rotation, the block's largest magnitude in registers, one 8-byte store of codes and one byte of scale (or one
// 32-byte store of bfloat16). Neighbouring threads own neighbouring tokens of one head, whose entries are neighbours in the page: codes
// and scales leave as whole sectors. Rotation: channel i < half with channel i + half, by the table row of the token's position
// counted from the row's start, x cos - y sin and y cos + x sin, rounded once to 32 bits, because a key next to a border of the 4-bit
// grid must fall on the side where the formula has it. Scale: max / 6 rounded to E4M3, code: x / scale rounded to E2M1,
// both quotients as IEEE rounds them, to nearest even.
// Bound: bytes at large sizes (4 read + 0.5625 or 2 written a value), launch latency at decode sizes.
//
// Read: the same split; a code times its scale is exact in bfloat16.
//
// Measured: 2.1 M positions of 4 heads of 64, bfloat16 665 us to append and 658 us to read (6.5 TB/s, the copy's rate), 4 bits 634 us (the
// rounding's instructions: 63% of the issue slots) and 457 us (6.0 TB/s); one token a row of 64 rows 9 us with a cold cache.
#include "paged.cuh"

namespace ghb {

constexpr int APPEND_THREADS = 256;
constexpr int ROWS_IN_SMEM = 1024;          // q_start entries kept in shared memory (beyond it: searched in global memory)

__device__ __forceinline__ const int* stage_q_start(const PagedRows& r, int* s) {
  // Out of order, the search may find no row for a token and never look at the row that is wrong: one CTA looks at all of them.
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < r.B; i += blockDim.x) { const int q = r.q_start[i], next = r.q_start[i + 1]; if (q < 0 || next < q || next > r.n) *r.err = ST_Q_START; }
  if (r.B + 1 > ROWS_IN_SMEM) return r.q_start;
  for (int i = threadIdx.x; i <= r.B; i += blockDim.x) s[i] = r.q_start[i];
  __syncthreads();
  return s;
}

// 32 bytes a lane and instruction: whole sectors
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7]) : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// 16 values as they lie in memory, and as float32
template <typename T> struct Raw16 { uint32_t w[4 * sizeof(T)]; };
template <typename T> __device__ __forceinline__ void load16(const T* p, Raw16<T>& r) {
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) load32(reinterpret_cast<const char*>(p) + 32 * i, r.w + 8 * i);
}
__device__ __forceinline__ void widen(const Raw16<float>& r, float* x) {
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(r.w[i]);
}
__device__ __forceinline__ void widen(const Raw16<__nv_bfloat16>& r, float* x) {
#pragma unroll
  for (int i = 0; i < 8; ++i) { x[2 * i] = __uint_as_float(r.w[i] << 16); x[2 * i + 1] = __uint_as_float(r.w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* x) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void load8(const float* p, float* x) {
  const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
  x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
}

// x c - y s and the like, rounded once: both products with what their rounding added (fused multiply-add), their sum with what its
// rounding added (Knuth's two-sum), the three taken off last. About 48 bits, in float32 instructions: conversions to 64 bits run at a
// sixteenth of their rate. (The remainders stand the other way round, taken off and not added: one that is zero is then +0, and a sum of -0 stays
// -0 without it.)
__device__ __forceinline__ float two_products(float a, float c, float b, float s) {
  const float p = __fmul_rn(a, c), q = __fmul_rn(b, s);
  const float ep = __fmaf_rn(-a, c, p), eq = __fmaf_rn(-b, s, q);
  const float sum = __fadd_rn(p, q), bb = __fadd_rn(sum, -p);
  const float es = __fadd_rn(__fadd_rn(__fadd_rn(sum, -bb), -p), __fadd_rn(bb, -q));
  const float r = __fadd_rn(sum, -__fadd_rn(es, __fadd_rn(ep, eq)));
  return isfinite(r) ? r : sum;          // (a remainder of an infinity is not a number)
}

// x[0 .. 16) at channels c0 .. of a head at `head`, rotated where they are rotary (half a multiple of 8) by the table's row at co, si.
template <typename T>
__device__ __forceinline__ void rotate16(const T* head, int c0, int half, const float* co, const float* si, float* x) {
#pragma unroll
  for (int g = 0; g < 16; g += 8) {
    const int c = c0 + g;
    if (c >= 2 * half) continue;
    const bool low = c < half;
    float y[8], cs[8], sn[8];
    load8(head + (low ? c + half : c - half), y);
    load8(co + (low ? c : c - half), cs);
    load8(si + (low ? c : c - half), sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[g + i] = two_products(x[g + i], cs[i], y[i], low ? -sn[i] : sn[i]);
  }
}

constexpr float LARGEST = 2688.f;          // 6 * 448

// a / b rounded as IEEE asks (Markstein's theorem: from the rounded reciprocal, one correction by the exact remainder), so that a
// value on a border of the grid falls where the division puts it. b is 2^-9 .. 448, |a| at most 2688.
__device__ __forceinline__ float quotient(float a, float b, float inv) {
  const float q = __fmul_rn(a, inv);
  return __fmaf_rn(__fmaf_rn(-q, b, a), inv, q);
}
// -a / b of two at once in the packed instructions: b twice, and minus its reciprocal twice. Negated, because the sum with a
// remainder of +0 then keeps the sign of a zero: for a = -0 it is +0 + -0, for a = +0 it is -0 + -0.
__device__ __forceinline__ uint64_t both(float lo, float hi) { uint64_t p; asm("mov.b64 %0, {%1, %2};" : "=l"(p) : "f"(lo), "f"(hi)); return p; }
__device__ __forceinline__ float2 minus_quotients(uint64_t a, uint64_t b, uint64_t ninv) {
  uint64_t q, r;
  float2 y;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(a), "l"(ninv));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(q), "l"(b), "l"(a));
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(r), "l"(ninv), "l"(q));
  asm("mov.b64 {%0, %1}, %2;" : "=f"(y.x), "=f"(y.y) : "l"(r));
  return y;
}

// 16 values -> 8 bytes of codes and the scale's byte.
__device__ __forceinline__ uint8_t quantize16(float* x, uint2& codes) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; i += 2) asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(x[i])), "f"(fabsf(x[i + 1])));
  if (!(top <= LARGEST)) {
    top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -LARGEST), LARGEST);
      top = fmaxf(top, fabsf(x[i]));
    }
  }
  const uint8_t sb = __nv_cvt_float_to_fp8(quotient(top, 6.f, 1.f / 6.f), __NV_SATFINITE, __NV_E4M3);
  const float s = e4m3_to_float(sb);
  uint32_t w[2] = {0u, 0u};
  if (s > 0.f) {
    const float ninv = -__frcp_rn(s);
    const uint64_t s2 = both(s, s), ninv2 = both(ninv, ninv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 y = minus_quotients(both(x[2 * i], x[2 * i + 1]), s2, ninv2);
      w[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(y, __NV_E2M1, cudaRoundNearest)) << (8 * (i & 3));
    }
    w[0] ^= 0x88888888u; w[1] ^= 0x88888888u;
  }
  codes = make_uint2(w[0], w[1]);
  return sb;
}

// Where a thread works: packed token j, its row and position, the entry of the position in head 0 (head h: h pages' slots further), or
// none. Looked up once for all the heads that the thread does. False: no row owns the token.
struct Spot { int b, t, start; long entry; };
__device__ __forceinline__ bool spot_of(const PagedRows& r, const int* qs, long j, Spot& s) {
  s.entry = -1;
  s.b = row_of(qs, r.B, static_cast<int>(j));
  if (s.b < 0) return false;             // padding
  const Row row = load_row(r, s.b);
  if (j < row.q0 || j >= row.q0 + row.nq) return false;          // (its range is refused)
  if (row.len == 0) return true;
  s.t = row.len - (row.q0 + row.nq - static_cast<int>(j));
  s.start = row.start;
  s.entry = entry_of(r, s.b, s.t, 0);
  return true;
}

// One thread: 16 channels (block blk) of one token, in the keys and values (2 Hkv of them) z0 .. z0 + per.
template <typename T, bool FP4>
__global__ void __launch_bounds__(APPEND_THREADS, 3) paged_append_kernel(PagedRows r, PagedPool c, const T* k, long k_ts, long k_hs, const T* v, long v_ts,
                                                                      long v_hs, const float* cos, const float* sin, int half, int n_pos, int per) {
  __shared__ int sqs[ROWS_IN_SMEM];
  const int* qs = stage_q_start(r, sqs);
  const int blocks = c.hd >> 4, b_log = __ffs(blocks) - 1;
  const long item = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int blk = static_cast<int>(item) & (blocks - 1);
  const long j = item >> b_log;
  if (j >= r.n) return;
  const int z0 = blockIdx.y * per, z1 = min(2 * r.Hkv, z0 + per);
  auto head_of = [&](int z) { return z >= r.Hkv ? v + j * v_ts + (z - r.Hkv) * v_hs : k + j * k_ts + z * k_hs; };
  constexpr int AHEAD = sizeof(T) == 2 && !FP4 ? 2 : 1;        // heads on their way together, as registers allow
  Raw16<T> raw[AHEAD];
  auto load = [&](int z) {
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load16(head_of(min(z + i, z1 - 1)) + blk * 16, raw[i]);
  };
  load(z0);        // under way during the look-ups
  Spot s;
  if (!spot_of(r, qs, j, s) || s.entry < 0) return;
  const bool turns = blk * 16 < 2 * half;
  if (half > 0) {                        // (for the values too: a token without a rotation is left out whole)
    const int p = s.t - s.start;
    if (p < 0 || p >= n_pos) { *r.err = p < 0 ? ST_START : ST_ROPE; return; }
    cos += static_cast<long>(p) * half;
    sin += static_cast<long>(p) * half;
  }
  for (int zz = z0; zz < z1; zz += AHEAD) {
    if (AHEAD > 1 && zz > z0) load(zz);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const int z = zz + i;
      if (z >= z1) break;
      const bool value = z >= r.Hkv;
      const int h = value ? z - r.Hkv : z;
      const long e = s.entry + (static_cast<long>(h) << r.page_shift);
      float x[16];
      widen(raw[i], x);
      if (AHEAD == 1 && z + 1 < z1) load(z + 1);        // while this one is rounded
      if (turns && !value) rotate16(head_of(z), blk * 16, half, cos, sin, x);
      if (FP4) {
        uint2 codes;
        const uint8_t sb = quantize16(x, codes);
        uint8_t* base = static_cast<uint8_t*>(value ? c.v : c.k);
        *reinterpret_cast<uint2*>(base + e * (c.hd >> 1) + blk * 8) = codes;
        (value ? c.v_scale : c.k_scale)[e * blocks + blk] = sb;
      } else {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const __nv_bfloat162 p2 = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&p2);
        }
        store32(static_cast<__nv_bfloat16*>(value ? c.v : c.k) + e * c.hd + blk * 16, w);
      }
    }
  }
}

template <bool FP4>
__global__ void __launch_bounds__(APPEND_THREADS) paged_read_kernel(PagedRows r, PagedPool c, __nv_bfloat16* ko, __nv_bfloat16* vo, int fill, int per) {
  __shared__ int sqs[ROWS_IN_SMEM];
  const int* qs = stage_q_start(r, sqs);
  const int blocks = c.hd >> 4, b_log = __ffs(blocks) - 1;
  const long item = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int blk = static_cast<int>(item) & (blocks - 1);
  const long j = item >> b_log;
  if (j >= r.n) return;
  Spot s;
  if (!spot_of(r, qs, j, s) && !fill) return;
  const int z0 = blockIdx.y * per, z1 = min(2 * r.Hkv, z0 + per);
#pragma unroll 2
  for (int z = z0; z < z1; ++z) {
    const bool value = z >= r.Hkv;
    const int h = value ? z - r.Hkv : z;
    __nv_bfloat16* o = (value ? vo : ko) + (j * r.Hkv + h) * c.hd + blk * 16;
    uint32_t w[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (s.entry < 0) { store32(o, w); continue; }
    const long e = s.entry + (static_cast<long>(h) << r.page_shift);
    if (FP4) {
      const uint8_t* base = static_cast<const uint8_t*>(value ? c.v : c.k);
      const uint2 codes = *reinterpret_cast<const uint2*>(base + e * (c.hd >> 1) + blk * 8);
      const float sc = e4m3_to_float((value ? c.v_scale : c.k_scale)[e * blocks + blk]);
      const uint32_t cw[2] = {codes.x, codes.y};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2 hv = __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>((cw[i >> 2] >> (8 * (i & 3))) & 0xff), __NV_E2M1));
        const float2 f = __half22float2(hv);
        const __nv_bfloat162 p2 = __floats2bfloat162_rn(f.x * sc, f.y * sc);
        w[i] = *reinterpret_cast<const uint32_t*>(&p2);
      }
    } else {
      load32(static_cast<const __nv_bfloat16*>(value ? c.v : c.k) + e * c.hd + blk * 16, w);
    }
    store32(o, w);
  }
}

namespace {
// The grid: CTAs over (token, 16-channel block), and over the 2 Hkv keys and values, `per` of them a thread: one where that leaves
// enough threads to fill the GPU (a decode step: latency), more where `ctas_sm` CTAs an SM remain, so that a thread's look-up of its row
// and page serves several blocks. Measured, per = 1 / the rule: 18k tokens of 2 heads of 128 appended in bfloat16 16.8 / 14.8 us
// (3 CTAs an SM reside), 72k tokens of 8 heads of 64 read back from 4 bits 56 / 42 us (more, smaller ones).
struct Grid { dim3 g; int per; bool ok; };
Grid grid_of(const PagedRows& r, int hd, int half, int ctas_sm) {
  const long x = (static_cast<long>(r.n) * (hd >> 4) + APPEND_THREADS - 1) / APPEND_THREADS;
  const long pairs = 2l * r.Hkv;
  long per = x * pairs / (148l * ctas_sm);
  per = per < 1 ? 1 : per > pairs ? pairs : per;
  const long y = (pairs + per - 1) / per;
  const bool ok = x <= 0x7fffffffL && y <= 65535 && (hd == 64 || hd == 128 || hd == 256) && half % 8 == 0 && 2 * half <= hd;
  return {dim3(static_cast<unsigned>(x), static_cast<unsigned>(y)), static_cast<int>(per), ok};
}
}  // namespace

int paged_append(const PagedRows& r, const PagedPool& c, const void* k, long k_ts, long k_hs, const void* v, long v_ts, long v_hs, bool f32,
                 const float* cos, const float* sin, int half, int n_pos, cudaStream_t st) {
  if (r.n == 0) return 0;
  const Grid g = grid_of(r, c.hd, half, 4);
  if (!g.ok) return 1;
#define GHB_APPEND(T, F) paged_append_kernel<T, F><<<g.g, APPEND_THREADS, 0, st>>>(r, c, static_cast<const T*>(k), k_ts, k_hs, static_cast<const T*>(v), v_ts, v_hs, cos, sin, half, n_pos, g.per)
  if (f32) { if (c.fp4) GHB_APPEND(float, true); else GHB_APPEND(float, false); }
  else { if (c.fp4) GHB_APPEND(__nv_bfloat16, true); else GHB_APPEND(__nv_bfloat16, false); }
#undef GHB_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int paged_read(const PagedRows& r, const PagedPool& c, void* ko, void* vo, bool fill, cudaStream_t st) {
  if (r.n == 0) return 0;
  const Grid g = grid_of(r, c.hd, 0, 16);
  if (!g.ok) return 1;
  if (c.fp4) paged_read_kernel<true><<<g.g, APPEND_THREADS, 0, st>>>(r, c, static_cast<__nv_bfloat16*>(ko), static_cast<__nv_bfloat16*>(vo), fill, g.per);
  else paged_read_kernel<false><<<g.g, APPEND_THREADS, 0, st>>>(r, c, static_cast<__nv_bfloat16*>(ko), static_cast<__nv_bfloat16*>(vo), fill, g.per);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace ghb
