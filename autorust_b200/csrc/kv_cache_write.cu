// Writing the 8-bit key/value cache and reading it back (include/ar_attn.h, ar_kv_cache_append and ar_kv_cache_read).
//
//   write   a = max |x| over the call's tokens of a page and head;  s1 = a / 127, or the least 2^k >= a / 448;
//           s = s1, or max(s0, s1) on a page that holds earlier tokens;  code = rn(x * (1 / s)), earlier codes rn(code * (s0 / s))
//   read    x = code * s (+ mean)
//
// Both are bound by memory: (1 + element size) bytes per value.  One CTA owns one page of one head, so that nothing is
// shared between CTAs: the page's tokens are loaded once, 32 values per thread, and stay in registers between the maximum and the
// codes.  K and V are the two halves of grid.z.
#include <cuda_bf16.h>

#include "kv_cache.cuh"

namespace ar {
namespace {

constexpr int PER_THREAD = 32;              // values per thread
constexpr int VECS = PER_THREAD / 8;        // in vectors of 8
constexpr float SCALE_FLOOR = 8.673617379884035e-19f;  // 2^-60: an empty or all-zero page needs no case of its own

template <bool F32>
__device__ __forceinline__ void load8(const void* base, long long at, float (&x)[8]) {
  if constexpr (F32) {
    const float4* p = (const float4*)((const float*)base + at);
    const float4 a = p[0], b = p[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 w = *(const uint4*)((const __nv_bfloat16*)base + at);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = __uint_as_float(u[i] << 16);
      x[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
    }
  }
}
template <bool F32>
__device__ __forceinline__ void store8(void* base, long long at, const float (&x)[8]) {
  if constexpr (F32) {
    float4* p = (float4*)((float*)base + at);
    p[0] = make_float4(x[0], x[1], x[2], x[3]);
    p[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 w;
    __nv_bfloat162* h = (__nv_bfloat162*)&w;
#pragma unroll
    for (int i = 0; i < 4; i++) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *(uint4*)((__nv_bfloat16*)base + at) = w;
  }
}

// Codes of 8 values that are already divided by the scale; `dead` (a NaN scale): zeros, since the codes of a page must stay
// finite for the products of rows that do not see it.
__device__ __forceinline__ uint2 encode8(const float (&y)[8], int e4m3, bool dead) {
  uint32_t w[2] = {0u, 0u};
  if (!dead) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      uint32_t two;
      if (e4m3) {
        two = e4m3_codes(y[i], y[i + 1]);
      } else {
        const int a = max(-127, min(127, __float2int_rn(y[i]))), b = max(-127, min(127, __float2int_rn(y[i + 1])));
        two = (uint32_t)(a & 0xff) | ((uint32_t)(b & 0xff) << 8);
      }
      w[i >> 2] |= two << ((i & 2) * 8);
    }
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void decode8(const uint2& w, int e4m3, float (&x)[8]) {
#pragma unroll
  for (int i = 0; i < 8; i++) x[i] = kv_value(((i < 4 ? w.x : w.y) >> ((i & 3) * 8)) & 0xffu, e4m3);
}

// The scale of a largest magnitude given by its bits (infinities and NaN are the largest patterns).
__device__ __forceinline__ float scale_of(uint32_t bits, int e4m3) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if (!e4m3) return fmaxf(__uint_as_float(bits) / 127.0f, SCALE_FLOOR);
  // amax = 1.m * 2^e <= 448 * 2^k = 1.75 * 2^(8 + k); a subnormal amax is far below the floor
  const int e = (int)(bits >> 23) - 127;
  const int k = max(e - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -60);
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// E values of a page and head, E / 32 threads.
template <int E, bool F32>
__global__ void __launch_bounds__(E / PER_THREAD)
kv_append_kernel(const KvPool pool, const KvBatch batch, const KvRows kr, const KvRows vr) {
  constexpr int THREADS = E / PER_THREAD;
  const int page_tokens = 1 << pool.page_log2;
  const int d_log2 = pool.D == 128 ? 7 : 6;
  const KvPlace p = kv_place(batch, blockIdx.x, 1, pool.page_log2, 2);
  const int first = max(p.length - p.n, 0);            // position of the first token that is written
  const int skipped = max(p.n - p.length, 0);          // padding rows in front of it (negative positions)
  const int count = p.n - skipped;
  if (p.tile < 0 || count <= 0) return;
  const int blk = (first >> pool.page_log2) + p.tile;  // block of the sequence
  const long long at0 = (long long)blk << pool.page_log2;                         // its first token
  const int t0 = (int)max((long long)first - at0, 0ll);                           // rows of the page before the first new token
  const int t1 = (int)min((long long)first + count - at0, (long long)page_tokens);  // and up to the last
  if (t1 <= t0) return;
  const int h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const int page = kv_page(pool, batch, p.b, blk);
  if (page < 0) {
    if (threadIdx.x == 0) kv_report(batch);
    return;
  }
  const KvRows& rows = is_v ? vr : kr;
  uint8_t* codes = (is_v ? pool.v : pool.k) + ((long long)page * pool.Hkv + h) * E;
  float* scale_at = (is_v ? pool.v_scale : pool.k_scale) + (long long)page * pool.Hkv + h;
  const float s0 = t0 > 0 ? *scale_at : 0.0f;
  const float* mean = !is_v && pool.k_mean ? pool.k_mean + h * pool.D : nullptr;
  const long long row0 = p.row0 + skipped + (at0 - first);  // packed row of the page's row 0

  float x[VECS][8];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int e = (i * THREADS + threadIdx.x) * 8, t = e >> d_log2, d = e & (pool.D - 1);
    if (t >= t0 && t < t1) {
      load8<F32>(rows.p, (row0 + t) * rows.st + (long long)h * rows.sh + d, x[i]);
      if (mean) {
#pragma unroll
        for (int c = 0; c < 8; c++) x[i][c] -= mean[d + c];
      }
#pragma unroll
      for (int c = 0; c < 8; c++) top = max(top, __float_as_uint(x[i][c]) & 0x7fffffffu);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (THREADS > 32) {
    __shared__ uint32_t tops[THREADS / 32];
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < THREADS / 32; i++) top = max(top, tops[i]);
  } else {
    __syncwarp();
  }
  float s = scale_of(top, pool.e4m3);
  if (t0 > 0 && !(s > s0) && s == s) s = s0;  // (a NaN on either side stays)
  const bool dead = s != s;
  const float inverse = 1.0f / s;
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int e = (i * THREADS + threadIdx.x) * 8, t = e >> d_log2;
    if (t >= t0 && t < t1) {
      float y[8];
#pragma unroll
      for (int c = 0; c < 8; c++) y[c] = x[i][c] * inverse;
      *(uint2*)(codes + e) = encode8(y, pool.e4m3, dead);
    }
  }
  if (t0 > 0 && s > s0) {  // the scale has grown: the earlier codes move to it
    const float ratio = s0 / s;
    for (int e = threadIdx.x * 8; e < (t0 << d_log2); e += THREADS * 8) {
      float y[8];
      decode8(*(const uint2*)(codes + e), pool.e4m3, y);
#pragma unroll
      for (int c = 0; c < 8; c++) y[c] *= ratio;
      *(uint2*)(codes + e) = encode8(y, pool.e4m3, false);
    }
  }
  if (threadIdx.x == 0) *scale_at = s;
}

template <int E, bool F32>
__global__ void __launch_bounds__(E / PER_THREAD)
kv_read_kernel(const KvPool pool, const KvBatch batch, const KvRows kr, const KvRows vr) {
  constexpr int THREADS = E / PER_THREAD;
  const int page_tokens = 1 << pool.page_log2;
  const int d_log2 = pool.D == 128 ? 7 : 6;
  const KvPlace p = kv_place(batch, blockIdx.x, 1, pool.page_log2, 2);
  if (p.tile < 0 || p.n <= 0) return;
  const int first = max(p.length - p.n, 0);
  const int skipped = max(p.n - p.length, 0);
  const int count = p.n - skipped;
  const int h = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const KvRows& rows = is_v ? vr : kr;
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (p.tile == 0) {  // padding rows
    for (long long e = threadIdx.x * 8; e < ((long long)skipped << d_log2); e += THREADS * 8)
      store8<F32>(rows.p, (p.row0 + (e >> d_log2)) * rows.st + (long long)h * rows.sh + (e & (pool.D - 1)), zero);
  }
  const int blk = (first >> pool.page_log2) + p.tile;
  const long long at0 = (long long)blk << pool.page_log2;
  const int t0 = (int)max((long long)first - at0, 0ll);
  const int t1 = (int)min((long long)first + count - at0, (long long)page_tokens);
  if (t1 <= t0) return;
  const int page = kv_page(pool, batch, p.b, blk);
  if (page < 0 && threadIdx.x == 0) kv_report(batch);
  const uint8_t* codes = (is_v ? pool.v : pool.k) + ((long long)max(page, 0) * pool.Hkv + h) * E;
  const float s = (is_v ? pool.v_scale : pool.k_scale)[(long long)max(page, 0) * pool.Hkv + h];
  const float* mean = !is_v && pool.k_mean ? pool.k_mean + h * pool.D : nullptr;
  const long long row0 = p.row0 + skipped + (at0 - first);
  uint2 w[VECS];
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int e = (i * THREADS + threadIdx.x) * 8, t = e >> d_log2;
    if (t >= t0 && t < t1) w[i] = *(const uint2*)(codes + e);
  }
#pragma unroll
  for (int i = 0; i < VECS; i++) {
    const int e = (i * THREADS + threadIdx.x) * 8, t = e >> d_log2, d = e & (pool.D - 1);
    if (t >= t0 && t < t1) {
      float x[8];
      decode8(w[i], pool.e4m3, x);
#pragma unroll
      for (int c = 0; c < 8; c++) x[c] = page < 0 ? 0.f : x[c] * s;
      if (mean && page >= 0) {
#pragma unroll
        for (int c = 0; c < 8; c++) x[c] = __fadd_rn(x[c], mean[d + c]);  // (not contracted: the definition rounds the product)
      }
      store8<F32>(rows.p, (row0 + t) * rows.st + (long long)h * rows.sh + d, x);
    }
  }
}

template <bool WRITE, bool F32>
cudaError_t launch(const KvPool& pool, const KvBatch& batch, const KvRows& k, const KvRows& v, cudaStream_t stream) {
  const dim3 grid((unsigned)kv_places(batch.B, batch.T, 1, pool.page_log2, 2), (unsigned)pool.Hkv, 2);
  auto go = [&](auto kern, int E) {
    kern<<<grid, E / PER_THREAD, 0, stream>>>(pool, batch, k, v);
    return cudaGetLastError();
  };
#define AR_KV_E(E) (WRITE ? go(kv_append_kernel<E, F32>, E) : go(kv_read_kernel<E, F32>, E))
  switch (pool.D << pool.page_log2) {
    case 1024: return AR_KV_E(1024);
    case 2048: return AR_KV_E(2048);
    case 4096: return AR_KV_E(4096);
    case 8192: return AR_KV_E(8192);
    case 16384: return AR_KV_E(16384);
  }
#undef AR_KV_E
  return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_kv_append(const KvPool& pool, const KvBatch& batch, int dtype, const KvRows& k, const KvRows& v,
                             cudaStream_t stream) {
  return dtype == 0 ? launch<true, true>(pool, batch, k, v, stream) : launch<true, false>(pool, batch, k, v, stream);
}
cudaError_t launch_kv_read(const KvPool& pool, const KvBatch& batch, int dtype, const KvRows& k, const KvRows& v,
                           cudaStream_t stream) {
  return dtype == 0 ? launch<false, true>(pool, batch, k, v, stream) : launch<false, false>(pool, batch, k, v, stream);
}

}  // namespace ar
