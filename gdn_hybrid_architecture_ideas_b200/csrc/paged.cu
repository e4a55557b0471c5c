// Appending to and reading from a paged key/value cache in bfloat16 or 4 bits (layout and checks: paged.cuh).
//
// Append: one thread owns 16 consecutive channels (one 4-bit block) of one token's key or value head: two 16-byte loads,
// the rotation, the block's largest magnitude in registers, one 8-byte store of codes and one byte of scale (or two
// 16-byte stores of bfloat16). Rotation: channel i < half with channel i + half, by the table row of the token's position
// counted from the row's start, x cos - y sin and y cos + x sin. It runs in 64 bits (the products of a float32 and a
// 24-bit table entry are exact there, so each channel is rounded once, to 32 bits), because a key next to a border of
// the 4-bit grid must fall on the side where the formula has it; 3 such operations a rotary channel are hidden behind
// the loads. Scale: max / 6 rounded to E4M3, code: x / scale rounded to E2M1, both IEEE divisions, to nearest even.
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

template <typename T> __device__ __forceinline__ void load16(const T* p, float* x);
template <> __device__ __forceinline__ void load16<__nv_bfloat16>(const __nv_bfloat16* p, float* x) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    const uint4 u = reinterpret_cast<const uint4*>(p)[c];
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      x[c * 8 + 2 * i] = f.x; x[c * 8 + 2 * i + 1] = f.y;
    }
  }
}
template <> __device__ __forceinline__ void load16<float>(const float* p, float* x) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const float4 u = reinterpret_cast<const float4*>(p)[c];
    x[c * 4] = u.x; x[c * 4 + 1] = u.y; x[c * 4 + 2] = u.z; x[c * 4 + 3] = u.w;
  }
}

// x[0 .. 16) at channels c0 .. of a head at `head`: rotated where they are rotary (half a multiple of 8).
template <typename T>
__device__ __forceinline__ void rotate16(const T* head, int c0, int half, const float* cos, const float* sin, float* x) {
#pragma unroll
  for (int g = 0; g < 16; g += 8) {
    const int c = c0 + g;
    if (c >= 2 * half) continue;
    const bool lowside = c < half;
    const int at = lowside ? c : c - half;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const double co = cos[at + i], si = sin[at + i];
      const double y = static_cast<double>(static_cast<float>(head[lowside ? c + half + i : c - half + i]));
      const double a = static_cast<double>(x[g + i]);
      x[g + i] = static_cast<float>(lowside ? a * co - y * si : a * co + y * si);
    }
  }
}

// 16 values -> 8 bytes of codes and the scale's byte.
__device__ __forceinline__ uint8_t quantize16(float* x, uint2& codes) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = x[i] != x[i] ? 0.f : fminf(fmaxf(x[i], -2688.f), 2688.f);
    top = fmaxf(top, fabsf(x[i]));
  }
  const uint8_t sb = __nv_cvt_float_to_fp8(__fdiv_rn(top, 6.f), __NV_SATFINITE, __NV_E4M3);
  const float s = e4m3_to_float(sb);
  uint32_t w[2] = {0u, 0u};
  if (s > 0.f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 y = make_float2(__fdiv_rn(x[2 * i], s), __fdiv_rn(x[2 * i + 1], s));
      w[i >> 2] |= static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(y, __NV_E2M1, cudaRoundNearest)) << (8 * (i & 3));
    }
  }
  codes = make_uint2(w[0], w[1]);
  return sb;
}

template <typename T, bool FP4>
__global__ void __launch_bounds__(APPEND_THREADS) paged_append_kernel(PagedRows r, PagedPool c, const T* k, long k_ts, long k_hs, const T* v, long v_ts,
                                                                      long v_hs, const float* cos, const float* sin, int half, int n_pos) {
  __shared__ int sqs[ROWS_IN_SMEM];
  const int* qs = stage_q_start(r, sqs);
  const int blocks = c.hd >> 4;
  const long item = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int blk = static_cast<int>(item % blocks);
  const long rest = item / blocks;
  const int h = static_cast<int>(rest % r.Hkv);
  const long j = rest / r.Hkv;
  if (j >= r.n) return;
  const int b = row_of(qs, r.B, static_cast<int>(j));
  if (b < 0) return;
  const Row row = load_row(r, b);
  if (row.len == 0 || j < row.q0 || j >= row.q0 + row.nq) return;
  const int t = row.len - (row.q0 + row.nq - static_cast<int>(j));
  const long e = entry_of(r, b, t, h);
  if (e < 0) return;
  const bool value = blockIdx.y == 1;
  const T* head = value ? v + j * v_ts + h * v_hs : k + j * k_ts + h * k_hs;
  float x[16];
  load16(head + blk * 16, x);
  if (!value && half > 0) {
    const int p = t - row.start;
    if (p < 0 || p >= n_pos) { *r.err = p < 0 ? ST_START : ST_ROPE; return; }
    rotate16(head, blk * 16, half, cos + static_cast<long>(p) * half, sin + static_cast<long>(p) * half, x);
  }
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

template <bool FP4>
__global__ void __launch_bounds__(APPEND_THREADS) paged_read_kernel(PagedRows r, PagedPool c, __nv_bfloat16* ko, __nv_bfloat16* vo, int fill) {
  __shared__ int sqs[ROWS_IN_SMEM];
  const int* qs = stage_q_start(r, sqs);
  const int blocks = c.hd >> 4;
  const long item = static_cast<long>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int blk = static_cast<int>(item % blocks);
  const long rest = item / blocks;
  const int h = static_cast<int>(rest % r.Hkv);
  const long j = rest / r.Hkv;
  if (j >= r.n) return;
  const bool value = blockIdx.y == 1;
  uint4* o = reinterpret_cast<uint4*>((value ? vo : ko) + (j * r.Hkv + h) * c.hd + blk * 16);
  const int b = row_of(qs, r.B, static_cast<int>(j));
  long e = -1;
  if (b >= 0) {
    const Row row = load_row(r, b);
    if (row.len > 0 && j >= row.q0 && j < row.q0 + row.nq) e = entry_of(r, b, row.len - (row.q0 + row.nq - static_cast<int>(j)), h);
  } else if (!fill) {
    return;
  }
  if (e < 0) { o[0] = make_uint4(0, 0, 0, 0); o[1] = make_uint4(0, 0, 0, 0); return; }
  if (FP4) {
    const uint8_t* base = static_cast<const uint8_t*>(value ? c.v : c.k);
    const uint2 codes = *reinterpret_cast<const uint2*>(base + e * (c.hd >> 1) + blk * 8);
    const float s = e4m3_to_float((value ? c.v_scale : c.k_scale)[e * blocks + blk]);
    const uint32_t cw[2] = {codes.x, codes.y};
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2 hv = __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>((cw[i >> 2] >> (8 * (i & 3))) & 0xff), __NV_E2M1));
      const float2 f = __half22float2(hv);
      const __nv_bfloat162 p2 = __floats2bfloat162_rn(f.x * s, f.y * s);
      w[i] = *reinterpret_cast<const uint32_t*>(&p2);
    }
    o[0] = make_uint4(w[0], w[1], w[2], w[3]);
    o[1] = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(value ? c.v : c.k) + e * c.hd + blk * 16);
    const uint4 a = s[0], b4 = s[1];
    o[0] = a; o[1] = b4;
  }
}

namespace {
// blocks for n tokens x heads x 16-channel blocks; 0 where there is nothing to do or the grid would not hold it
long append_grid(const PagedRows& r, int hd) { return (static_cast<long>(r.n) * r.Hkv * (hd >> 4) + APPEND_THREADS - 1) / APPEND_THREADS; }
}  // namespace

int paged_append(const PagedRows& r, const PagedPool& c, const void* k, long k_ts, long k_hs, const void* v, long v_ts, long v_hs, bool f32,
                 const float* cos, const float* sin, int half, int n_pos, cudaStream_t st) {
  const long g = append_grid(r, c.hd);
  if (g == 0) return 0;
  if (g > 0x7fffffffL || c.hd % 16 || half % 8 || 2 * half > c.hd) return 1;
  const dim3 grid(static_cast<unsigned>(g), 2);
#define GHB_APPEND(T, F) paged_append_kernel<T, F><<<grid, APPEND_THREADS, 0, st>>>(r, c, static_cast<const T*>(k), k_ts, k_hs, static_cast<const T*>(v), v_ts, v_hs, cos, sin, half, n_pos)
  if (f32) { if (c.fp4) GHB_APPEND(float, true); else GHB_APPEND(float, false); }
  else { if (c.fp4) GHB_APPEND(__nv_bfloat16, true); else GHB_APPEND(__nv_bfloat16, false); }
#undef GHB_APPEND
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

int paged_read(const PagedRows& r, const PagedPool& c, void* ko, void* vo, bool fill, cudaStream_t st) {
  const long g = append_grid(r, c.hd);
  if (g == 0) return 0;
  if (g > 0x7fffffffL || c.hd % 16) return 1;
  const dim3 grid(static_cast<unsigned>(g), 2);
  if (c.fp4) paged_read_kernel<true><<<grid, APPEND_THREADS, 0, st>>>(r, c, static_cast<__nv_bfloat16*>(ko), static_cast<__nv_bfloat16*>(vo), fill);
  else paged_read_kernel<false><<<grid, APPEND_THREADS, 0, st>>>(r, c, static_cast<__nv_bfloat16*>(ko), static_cast<__nv_bfloat16*>(vo), fill);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace ghb
