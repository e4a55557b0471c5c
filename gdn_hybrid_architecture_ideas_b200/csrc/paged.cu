// Appending to and reading from a paged key/value cache in bfloat16 or 4 bits (layout and checks: paged.cuh).
//
// Append: one thread owns 16 consecutive channels (one 4-bit block) of one token, in one key or value head or in several: two 16-byte
// loads, the rotation, the block's largest magnitude in registers, one 8-byte store of codes and one byte of scale (or two
// 16-byte stores of bfloat16). Neighbouring threads own neighbouring tokens of one head, whose entries are neighbours in the page: codes
// and scales leave as whole sectors. Rotation: channel i < half with channel i + half, by the table row of the token's position
// counted from the row's start, x cos - y sin and y cos + x sin, rounded once to 32 bits, because a key next to a border of the 4-bit
// grid must fall on the side where the formula has it. Scale: max / 6 rounded to E4M3, code: x / scale rounded to E2M1,
// both quotients as IEEE rounds them, to nearest even.
// Bound: bytes at large sizes (4 read + 0.5625 or 2 written a value), launch latency at decode sizes.
//
// Read: the same split; a code times its scale is exact in bfloat16.
#include "paged.cuh"

namespace ghb {

constexpr int APPEND_THREADS = 256;
constexpr int ROWS_IN_SMEM = 1024;          // q_start entries kept in shared memory (beyond it: searched in global memory)

__device__ __forceinline__ const int* stage_q_start(const PagedRows& r, int* s) {
  if (r.B + 1 > ROWS_IN_SMEM) return r.q_start;
  for (int i = threadIdx.x; i <= r.B; i += blockDim.x) s[i] = r.q_start[i];
  __syncthreads();
  return s;
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float* x) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
    x[2 * i] = f.x; x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float* x) {
  const float4 u = reinterpret_cast<const float4*>(p)[0], v = reinterpret_cast<const float4*>(p)[1];
  x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
}

// x c - y s and the like, rounded once: both products with their exact remainders (fused multiply-add), their sum with its remainder
// (Knuth's two-sum), the remainders added last. About 48 bits, in float32 instructions: conversions to 64 bits run at a
// sixteenth of their rate.
__device__ __forceinline__ float two_products(float a, float c, float b, float s) {
  const float p = __fmul_rn(a, c), q = __fmul_rn(b, s);
  const float ep = __fmaf_rn(a, c, -p), eq = __fmaf_rn(b, s, -q);
  const float sum = __fadd_rn(p, q), bb = __fadd_rn(sum, -p);
  const float es = __fadd_rn(__fadd_rn(p, -__fadd_rn(sum, -bb)), __fadd_rn(q, -bb));
  const float r = __fadd_rn(sum, __fadd_rn(es, __fadd_rn(ep, eq)));
  return isfinite(r) ? r : sum;          // (a remainder of an infinity is not a number)
}

// x[0 .. 16) at channels c0 .. of a head at `head`, rotated where they are rotary (half a multiple of 8): co, si are the table's
// entries of these channels, the sine with the channel's sign.
template <typename T>
__device__ __forceinline__ void rotate16(const T* head, int c0, int half, const float* co, const float* si, float* x) {
#pragma unroll
  for (int g = 0; g < 16; g += 8) {
    const int c = c0 + g;
    if (c >= 2 * half) continue;
    float y[8];
    load8(head + (c < half ? c + half : c - half), y);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[g + i] = two_products(x[g + i], co[g + i], y[i], si[g + i]);
  }
}

constexpr float LARGEST = 2688.f;          // 6 * 448

// a / b rounded as IEEE asks (Markstein's theorem: from the rounded reciprocal, one correction by the exact remainder), so that a
// value on a border of the grid falls where the division puts it. b is 2^-9 .. 448, |a| at most 2688.
__device__ __forceinline__ float quotient(float a, float b, float inv) {
  const float q = __fmul_rn(a, inv);
  return __fmaf_rn(__fmaf_rn(-q, b, a), inv, q);
}

// 16 values -> 8 bytes of codes and the scale's byte.
__device__ __forceinline__ uint8_t quantize16(float* x, uint2& codes) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(x[i])));
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
    const float inv = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 y = make_float2(quotient(x[2 * i], s, inv), quotient(x[2 * i + 1], s, inv));
      w[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(y, __NV_E2M1, cudaRoundNearest)) << (8 * (i & 3));
    }
  }
  codes = make_uint2(w[0], w[1]);
  return sb;
}

// Where a thread works: packed token j, its row and position, the entry of the position in head 0 (head h: h pages' slots further), or
// none. Looked up once for all the heads that the thread does.
struct Spot { long j; int b, t, start; long entry; };
__device__ __forceinline__ bool spot_of(const PagedRows& r, const int* qs, long j, Spot& s) {
  s.j = j;
  s.entry = -1;
  s.b = row_of(qs, r.B, static_cast<int>(j));
  if (s.b < 0) return false;             // padding
  const Row row = load_row(r, s.b);
  if (row.len == 0 || j < row.q0 || j >= row.q0 + row.nq) return true;
  s.t = row.len - (row.q0 + row.nq - static_cast<int>(j));
  s.start = row.start;
  s.entry = entry_of(r, s.b, s.t, 0);
  return true;
}

// One thread: 16 channels (block blk) of one token, in the keys and values (2 Hkv of them) z0 .. z0 + per.
template <typename T, bool FP4>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(PagedRows r, PagedPool c, const T* k, long k_ts, long k_hs, const T* v, long v_ts,
                                                                      long v_hs, const float* cos, const float* sin, int half, int n_pos, int per) {
  __shared__ int sqs[ROWS_IN_SMEM];
  const int* qs = stage_q_start(r, sqs);
  const int blocks = c.hd >> 4, b_log = __ffs(blocks) - 1;
  const long item = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int blk = static_cast<int>(item) & (blocks - 1);
  const long j = item >> b_log;
  if (j >= r.n) return;
  Spot s;
  if (!spot_of(r, qs, j, s) || s.entry < 0) return;
  const int z0 = blockIdx.y * per, z1 = min(2 * r.Hkv, z0 + per);
  const bool turns = blk * 16 < 2 * half && z0 < r.Hkv;
  float co[16], si[16];
  if (half > 0 && z0 < r.Hkv) {
    const int p = s.t - s.start;
    if (p < 0 || p >= n_pos) { *r.err = p < 0 ? ST_START : ST_ROPE; return; }
    if (turns) {
#pragma unroll
      for (int g = 0; g < 16; g += 8) {
        const int ch = blk * 16 + g, at = ch < half ? ch : ch - half;
        if (ch >= 2 * half) continue;
        load8(cos + static_cast<long>(p) * half + at, co + g);
        load8(sin + static_cast<long>(p) * half + at, si + g);
#pragma unroll
        for (int i = 0; i < 8; ++i) si[g + i] = ch < half ? -si[g + i] : si[g + i];
      }
    }
  }
  for (int z = z0; z < z1; ++z) {
    const bool value = z >= r.Hkv;
    const int h = value ? z - r.Hkv : z;
    const T* head = value ? v + j * v_ts + h * v_hs : k + j * k_ts + h * k_hs;
    const long e = s.entry + (static_cast<long>(h) << r.page_shift);
    float x[16];
    load8(head + blk * 16, x);
    load8(head + blk * 16 + 8, x + 8);
    if (turns && !value) rotate16(head, blk * 16, half, co, si, x);
    if (FP4) {
      uint2 codes;
      const uint8_t sb = quantize16(x, codes);
      uint8_t* base = static_cast<uint8_t*>(value ? c.v : c.k);
      *reinterpret_cast<uint2*>(base + e * (c.hd >> 1) + blk * 8) = codes;
      (value ? c.v_scale : c.k_scale)[e * blocks + blk] = sb;
    } else {
      __nv_bfloat16* o = static_cast<__nv_bfloat16*>(value ? c.v : c.k) + e * c.hd + blk * 16;
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 p2 = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&p2);
      }
      reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
      reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
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
    uint4* o = reinterpret_cast<uint4*>((value ? vo : ko) + (j * r.Hkv + h) * c.hd + blk * 16);
    if (s.entry < 0) { o[0] = make_uint4(0, 0, 0, 0); o[1] = make_uint4(0, 0, 0, 0); continue; }
    const long e = s.entry + (static_cast<long>(h) << r.page_shift);
    if (FP4) {
      const uint8_t* base = static_cast<const uint8_t*>(value ? c.v : c.k);
      const uint2 codes = *reinterpret_cast<const uint2*>(base + e * (c.hd >> 1) + blk * 8);
      const float sc = e4m3_to_float((value ? c.v_scale : c.k_scale)[e * blocks + blk]);
      const uint32_t cw[2] = {codes.x, codes.y};
      uint32_t w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __half2 hv = __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>((cw[i >> 2] >> (8 * (i & 3))) & 0xff), __NV_E2M1));
        const float2 f = __half22float2(hv);
        const __nv_bfloat162 p2 = __floats2bfloat162_rn(f.x * sc, f.y * sc);
        w[i] = *reinterpret_cast<const uint32_t*>(&p2);
      }
      o[0] = make_uint4(w[0], w[1], w[2], w[3]);
      o[1] = make_uint4(w[4], w[5], w[6], w[7]);
    } else {
      const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(value ? c.v : c.k) + e * c.hd + blk * 16);
      const uint4 a = src[0], b4 = src[1];
      o[0] = a; o[1] = b4;
    }
  }
}

namespace {
// The grid: CTAs over (token, 16-channel block), and over the 2 Hkv keys and values, `per` of them a thread. One where that leaves
// enough threads to fill the GPU (a decode step: latency); as many as still do at large sizes, where a thread's look-up of its row and
// page costs as much as a block (81k tokens of 8 heads, 4 bits: append 126 us at one, NNN at all; reading back 56 and NNN).
struct Grid { dim3 g; int per; bool ok; };
Grid append_grid(const PagedRows& r, int hd, int half) {
  const long x = (static_cast<long>(r.n) * (hd >> 4) + APPEND_THREADS - 1) / APPEND_THREADS;
  const long pairs = 2l * r.Hkv;
  long per = x * pairs / (148l * 16);          // 16 CTAs an SM
  per = per < 1 ? 1 : per > pairs ? pairs : per;
  const long y = (pairs + per - 1) / per;
  const bool ok = x <= 0x7fffffffL && y <= 65535 && (hd == 64 || hd == 128 || hd == 256) && half % 8 == 0 && 2 * half <= hd;
  return {dim3(static_cast<unsigned>(x), static_cast<unsigned>(y)), static_cast<int>(per), ok};
}
}  // namespace

int paged_append(const PagedRows& r, const PagedPool& c, const void* k, long k_ts, long k_hs, const void* v, long v_ts, long v_hs, bool f32,
                 const float* cos, const float* sin, int half, int n_pos, cudaStream_t st) {
  if (r.n == 0) return 0;
  const Grid g = append_grid(r, c.hd, half);
  if (!g.ok) return 1;
#define GHB_APPEND(T, F) paged_append_kernel<T, F><<<g.g, APPEND_THREADS, 0, st>>>(r, c, static_cast<const T*>(k), k_ts, k_hs, static_cast<const T*>(v), v_ts, v_hs, cos, sin, half, n_pos, g.per)
  if (f32) { if (c.fp4) GHB_APPEND(float, true); else GHB_APPEND(float, false); }
  else { if (c.fp4) GHB_APPEND(__nv_bfloat16, true); else GHB_APPEND(__nv_bfloat16, false); }
#undef GHB_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int paged_read(const PagedRows& r, const PagedPool& c, void* ko, void* vo, bool fill, cudaStream_t st) {
  if (r.n == 0) return 0;
  const Grid g = append_grid(r, c.hd, 0);
  if (!g.ok) return 1;
  if (c.fp4) paged_read_kernel<true><<<g.g, APPEND_THREADS, 0, st>>>(r, c, static_cast<__nv_bfloat16*>(ko), static_cast<__nv_bfloat16*>(vo), fill, g.per);
  else paged_read_kernel<false><<<g.g, APPEND_THREADS, 0, st>>>(r, c, static_cast<__nv_bfloat16*>(ko), static_cast<__nv_bfloat16*>(vo), fill, g.per);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace ghb
