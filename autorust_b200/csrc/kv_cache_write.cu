// Writing the 8-bit key/value cache and reading it back (include/ar_attn.h, ar_kv_cache_append and ar_kv_cache_read).
//
//   write   a = max |x| over the call's tokens of a page and head;  s1 = a / 127, or the least 2^k >= a / 448;
//           s = s1, or max(s0, s1) on a page that holds earlier tokens;  code = rn(x * (1 / s)), earlier codes rn(code * (s0 / s))
//   read    x = code * s (+ mean)
//
// Both are bound by memory: (1 + element size) bytes per value.  One CTA owns one page of one head at a time, so that nothing is
// shared between CTAs: the page's tokens are loaded once, 32 values per thread, and stay in registers between the maximum and the
// codes.  Finding the sequence, its length and its page is a chain of dependent loads, about 2.5 us: in large calls a CTA takes
// several heads of its page one after the other, and asks for the next head's values before it works on this one's (writing: by
// cp.async into shared memory, which leaves registers for more threads).  K and V
// are the two halves of grid.z.
//
// Measured, bf16, 8 kv heads, D = 128, INT8: 32768 tokens written 44.4 us (4.5 TB/s), read back 38 (5.2 TB/s), 131072 tokens read back 139 (5.8 TB/s).
// Writing also waits for a page's maximum between its values and their codes.
#include <cuda_bf16.h>

#include "ar_ptx.cuh"
#include "kv_cache.cuh"

#include <algorithm>

namespace ar {
namespace {

constexpr int PER_THREAD = 32;              // values per thread
constexpr int VECS = PER_THREAD / 8;        // in vectors of 8
// Threads per SM that the writing kernel is built for (32768 tokens written: 49 us with 512, 45 with 768, 50 with 1024, which spill).
constexpr int APPEND_THREADS = 768;
constexpr float SCALE_FLOOR = 8.673617379884035e-19f;  // 2^-60: an empty or all-zero page needs no case of its own

// 8 values as they lie in memory.
template <bool F32>
struct Raw {
  uint4 w[F32 ? 2 : 1];
};
template <bool F32>
__device__ __forceinline__ void values8(const Raw<F32>& r, float (&x)[8]) {
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      x[4 * i] = __uint_as_float(r.w[i].x);
      x[4 * i + 1] = __uint_as_float(r.w[i].y);
      x[4 * i + 2] = __uint_as_float(r.w[i].z);
      x[4 * i + 3] = __uint_as_float(r.w[i].w);
    }
  } else {
    const uint32_t u[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
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

// Codes of 8 values that are already divided by the scale (and so inside +-127 or +-448); `dead` (a NaN scale): zeros, since the
// codes of a page must stay finite for the products of rows that do not see it.
template <bool E4M3>
__device__ __forceinline__ uint2 encode8(const float (&y)[8], bool dead) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float* v = y + 4 * i;
    if constexpr (E4M3) {
      w[i] = e4m3_codes(v[0], v[1]) | e4m3_codes(v[2], v[3]) << 16;
    } else {  // 1.5 * 2^23 + y, rounded to nearest even, has the code in its low byte
      float u[4];
#pragma unroll
      for (int c = 0; c < 4; c++) u[c] = __fadd_rn(v[c], 12582912.0f);
      w[i] = __byte_perm(__byte_perm(__float_as_uint(u[0]), __float_as_uint(u[1]), 0x0040),
                         __byte_perm(__float_as_uint(u[2]), __float_as_uint(u[3]), 0x0040), 0x5410);
    }
    if (dead) w[i] = 0u;
  }
  return make_uint2(w[0], w[1]);
}
template <bool E4M3>
__device__ __forceinline__ void decode8(const uint2& w, float (&x)[8]) {
  float lo[4], hi[4];
  kv_values4<E4M3>(w.x, lo);
  kv_values4<E4M3>(w.y, hi);
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[i] = lo[i];
    x[4 + i] = hi[i];
  }
}
// max(|a|, |b|, |c|), NaN if one is.
__device__ __forceinline__ float max_abs_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two values at a time.  (Sums of these products are taken one by one: a packed product and a packed sum behind it become one
// multiply-add, which rounds once where the definition rounds twice.)
__device__ __forceinline__ void scale8(const float (&x)[8], float by, float (&y)[8]) {
  const uint64_t by2 = arptx::pack_f32x2(by, by);
#pragma unroll
  for (int c = 0; c < 8; c += 2) arptx::unpack_f32x2(arptx::mul_f32x2(arptx::pack_f32x2(x[c], x[c + 1]), by2), y[c], y[c + 1]);
}

// The scale of a largest magnitude given by its bits (infinities and NaN are the largest patterns).
template <bool E4M3>
__device__ __forceinline__ float scale_of(uint32_t bits) {
  if (bits >= 0x7f800000u) return __uint_as_float(0x7fc00000u);
  if constexpr (!E4M3) return fmaxf(__uint_as_float(bits) / 127.0f, SCALE_FLOOR);
  // amax = 1.m * 2^e <= 448 * 2^k = 1.75 * 2^(8 + k); a subnormal amax is far below the floor
  const int e = (int)(bits >> 23) - 127;
  const int k = max(e - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -60);
  return __uint_as_float((uint32_t)(k + 127) << 23);
}

// What a CTA does: the rows [t0, t1) of a page, packed rows row0 + t.
struct Span {
  int page;         // -1: there is none (reported)
  int t0, t1;
  long long row0;
  int padding;      // read: this many of the sequence's rows, from pad_row on, have no token
  long long pad_row;
};
__device__ __forceinline__ Span span_of(const KvPool& pool, const KvBatch& batch) {
  const KvPlace p = kv_place(batch, blockIdx.x, 1, pool.page_log2, 2);
  Span s{-1, 0, 0, 0, 0, 0};
  if (p.tile < 0 || p.n <= 0) return s;
  const int first = max(p.length - p.n, 0);      // position of the first token
  const int skipped = max(p.n - p.length, 0);    // padding rows in front of it (negative positions)
  if (p.tile == 0) s.padding = skipped;
  s.pad_row = p.row0;
  const int blk = (first >> pool.page_log2) + p.tile;    // block of the sequence
  const long long at0 = (long long)blk << pool.page_log2;  // its first token
  s.t0 = (int)max((long long)first - at0, 0ll);
  s.t1 = (int)min((long long)first + (p.n - skipped) - at0, 1ll << pool.page_log2);
  s.row0 = p.row0 + skipped + (at0 - first);
  if (s.t1 > s.t0) {
    s.page = kv_page(pool, batch, p.b, blk);
    if (s.page < 0 && threadIdx.x == 0) kv_report(batch);
  }
  return s;
}

// E = page * D values of a page and head, E / 32 threads; heads blockIdx.y, blockIdx.y + gridDim.y, ...  A thread has the same 8 channels
// of every TOKENS-th token.
// The next head's values on their way: cp.async into places that only the thread which asks reads, so without barriers.  32768 tokens written: 44.4 us;
// with these values in registers 47.3, with a third stage 45.3, a fourth 46.3.
template <int E, bool F32>
struct Ring {
  static constexpr int STAGE = E * (F32 ? 4 : 2);
  static constexpr int BYTES = 2 * STAGE;
};
template <int E, int D, bool E4M3, bool F32>
__global__ void __launch_bounds__(E / PER_THREAD, (F32 ? 512 : APPEND_THREADS) * PER_THREAD / E)
kv_append_kernel(const KvPool pool, const KvBatch batch, const KvRows kr, const KvRows vr) {
  constexpr int THREADS = E / PER_THREAD, TOKENS = THREADS * 8 / D;
  __shared__ uint32_t tops[2][THREADS / 32];
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Span span = span_of(pool, batch);
  if (span.page < 0) return;
  const bool is_v = blockIdx.z != 0;
  const KvRows rows{is_v ? vr.p : kr.p, is_v ? vr.st : kr.st, is_v ? vr.sh : kr.sh};
  const int t = threadIdx.x * 8 / D, d = threadIdx.x * 8 % D;
  const long long first_row = (span.row0 + t) * rows.st + d, step = TOKENS * rows.st;
  bool in[VECS];
#pragma unroll
  for (int i = 0; i < VECS; i++) in[i] = t + i * TOKENS >= span.t0 && t + i * TOKENS < span.t1;
  uint8_t* codes = (is_v ? pool.v : pool.k) + (long long)span.page * pool.Hkv * E;
  float* scales = (is_v ? pool.v_scale : pool.k_scale) + (long long)span.page * pool.Hkv;
  const float* means = is_v ? nullptr : pool.k_mean;
  using R = Ring<E, F32>;
  constexpr int PER_VEC = F32 ? 2 : 1;
  extern __shared__ __align__(16) uint8_t ring[];
  uint8_t* const mine = ring + threadIdx.x * 16;
  auto fetch = [&](int h, int stage) {
    if (h < pool.Hkv) {
      const uint32_t to = arptx::smem_u32(mine) + stage * R::STAGE;
      const long long at = first_row + (long long)h * rows.sh;
#pragma unroll
      for (int i = 0; i < VECS; i++)
        if (in[i]) {
          const char* from = (const char*)rows.p + (at + i * step) * (F32 ? 4 : 2);
#pragma unroll
          for (int j = 0; j < PER_VEC; j++) arptx::cp_async16(to + (i * PER_VEC + j) * THREADS * 16, from + j * 16, true);
        }
    }
    arptx::cp_async_commit();
  };
  fetch(blockIdx.y, 0);
  for (int h = blockIdx.y, n = 0; h < pool.Hkv; h += gridDim.y, n ^= 1) {
    const float s0 = span.t0 > 0 ? scales[h] : 0.f;
    float x[VECS][8];
    float most = 0.f;
    float4 ma, mb;
    if (means) {
      ma = *(const float4*)(means + h * D + d);
      mb = *(const float4*)(means + h * D + d + 4);
    }
    fetch(h + gridDim.y, n ^ 1);  // (what was read there is in use by now)
    arptx::cp_async_wait<1>();
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      if (in[i]) {
        Raw<F32> raw;
#pragma unroll
        for (int j = 0; j < PER_VEC; j++) raw.w[j] = *(const uint4*)(mine + n * R::STAGE + (i * PER_VEC + j) * THREADS * 16);
        values8<F32>(raw, x[i]);
        if (means) {
          const float off[8] = {-ma.x, -ma.y, -ma.z, -ma.w, -mb.x, -mb.y, -mb.z, -mb.w};
#pragma unroll
          for (int c = 0; c < 8; c += 2)
            arptx::unpack_f32x2(arptx::add_f32x2(arptx::pack_f32x2(x[i][c], x[i][c + 1]), arptx::pack_f32x2(off[c], off[c + 1])), x[i][c],
                                x[i][c + 1]);
        }
#pragma unroll
        for (int c = 0; c < 8; c += 2) most = max_abs_nan(most, x[i][c], x[i][c + 1]);
      }
    }
    uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));  // (infinities and NaN are the largest patterns)
    if constexpr (THREADS > 32) {
      if ((threadIdx.x & 31) == 0) tops[n][threadIdx.x >> 5] = top;
      __syncthreads();  // (the other half of tops is written before the next one: no second barrier)
      top = __reduce_max_sync(0xffffffffu, tops[n][threadIdx.x & (THREADS / 32 - 1)]);
    } else {
      __syncwarp();
    }
    uint8_t* to = codes + (long long)h * E + threadIdx.x * 8;
    float s = scale_of<E4M3>(top);
    if (span.t0 > 0 && !(s > s0) && s == s) s = s0;  // (a NaN on either side stays)
    const bool dead = s != s;
    const float inverse = 1.0f / s;
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      if (in[i]) {
        float y[8];
        scale8(x[i], inverse, y);
        *(uint2*)(to + i * THREADS * 8) = encode8<E4M3>(y, dead);
      }
    }
    if (span.t0 > 0 && s > s0) {  // the scale has grown: the earlier codes move to it
      const float ratio = s0 / s;
#pragma unroll 1
      for (int i = 0; i < VECS; i++) {
        if (t + i * TOKENS >= span.t0) break;
        float y[8];
        decode8<E4M3>(*(const uint2*)(to + i * THREADS * 8), y);
        scale8(y, ratio, y);
        *(uint2*)(to + i * THREADS * 8) = encode8<E4M3>(y, false);
      }
    }
    if (threadIdx.x == 0) scales[h] = s;
  }
}

template <int E, int D, bool E4M3, bool F32>
__global__ void __launch_bounds__(E / PER_THREAD)
kv_read_kernel(const KvPool pool, const KvBatch batch, const KvRows kr, const KvRows vr) {
  constexpr int THREADS = E / PER_THREAD, TOKENS = THREADS * 8 / D;
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const Span span = span_of(pool, batch);
  const bool is_v = blockIdx.z != 0;
  const KvRows rows{is_v ? vr.p : kr.p, is_v ? vr.st : kr.st, is_v ? vr.sh : kr.sh};
  const int t = threadIdx.x * 8 / D, d = threadIdx.x * 8 % D;
  const float zero[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (span.padding > 0) {
    for (int h = blockIdx.y; h < pool.Hkv; h += gridDim.y)
      for (int r = t; r < span.padding; r += TOKENS) store8<F32>(rows.p, (span.pad_row + r) * rows.st + (long long)h * rows.sh + d, zero);
  }
  if (span.t1 <= span.t0) return;
  const long long first_row = (span.row0 + t) * rows.st + d, step = TOKENS * rows.st;
  bool in[VECS];
#pragma unroll
  for (int i = 0; i < VECS; i++) in[i] = t + i * TOKENS >= span.t0 && t + i * TOKENS < span.t1;
  if (span.page < 0) {  // reported
    for (int h = blockIdx.y; h < pool.Hkv; h += gridDim.y)
#pragma unroll
      for (int i = 0; i < VECS; i++)
        if (in[i]) store8<F32>(rows.p, first_row + i * step + (long long)h * rows.sh, zero);
    return;
  }
  const uint8_t* codes = (is_v ? pool.v : pool.k) + (long long)span.page * pool.Hkv * E + threadIdx.x * 8;
  const float* scales = (is_v ? pool.v_scale : pool.k_scale) + (long long)span.page * pool.Hkv;
  const float* means = is_v ? nullptr : pool.k_mean;
  uint2 w[VECS];
  float next_s = 0.f;
  auto fetch = [&](int h) {
    if (h >= pool.Hkv) return;
    next_s = scales[h];
#pragma unroll
    for (int i = 0; i < VECS; i++)
      if (in[i]) w[i] = *(const uint2*)(codes + (long long)h * E + i * THREADS * 8);
  };
  fetch(blockIdx.y);
  for (int h = blockIdx.y; h < pool.Hkv; h += gridDim.y) {
    const float s = next_s;
    float mean[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (means) {
      const float4 a = *(const float4*)(means + h * D + d), b = *(const float4*)(means + h * D + d + 4);
      mean[0] = a.x; mean[1] = a.y; mean[2] = a.z; mean[3] = a.w;
      mean[4] = b.x; mean[5] = b.y; mean[6] = b.z; mean[7] = b.w;
    }
    uint2 now[VECS];
#pragma unroll
    for (int i = 0; i < VECS; i++) now[i] = w[i];
    fetch(h + gridDim.y);
#pragma unroll
    for (int i = 0; i < VECS; i++) {
      if (in[i]) {
        float x[8];
        decode8<E4M3>(now[i], x);
        scale8(x, s, x);
        if (means) {
#pragma unroll
          for (int c = 0; c < 8; c++) x[c] = __fadd_rn(x[c], mean[c]);
        }
        store8<F32>(rows.p, first_row + i * step + (long long)h * rows.sh, x);
      }
    }
  }
}

// CTAs up to which every head of a page gets one of its own: 8 per SM (4 of prompts of up to 789 tokens written and read back: 5.7 + 4.1 us,
// with 4 per SM 7.3 + 4.5; 32768 tokens 44.4 + 39 and 44.6 + 40.4; 12 per SM like 8).
constexpr int SPREAD_CTAS = 8 * 148;

template <bool WRITE, bool E4M3, bool F32>
cudaError_t launch(const KvPool& pool, const KvBatch& batch, const KvRows& k, const KvRows& v, cudaStream_t stream) {
  const long long places = kv_places(batch, 1, pool.page_log2, 2);
  const long long per_cta = std::max(1ll, std::min((long long)pool.Hkv, places * pool.Hkv * 2 / SPREAD_CTAS));  // heads
  const dim3 grid((unsigned)places, (unsigned)((pool.Hkv + per_cta - 1) / per_cta), 2);
  auto go = [&](auto kern, int E, int smem) {
    if (smem > 47 * 1024) {  // (48 KB with the static part)
      const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
      if (e != cudaSuccess) return e;
    }
    return launch_early(kern, grid, dim3(E / PER_THREAD), smem, stream, pool, batch, k, v);
  };
#define AR_KV_E(E, D) (WRITE ? go(kv_append_kernel<E, D, E4M3, F32>, E, Ring<E, F32>::BYTES) : go(kv_read_kernel<E, D, E4M3, F32>, E, 0))
  if (pool.D == 128) {
    switch (pool.page_log2) {
      case 4: return AR_KV_E(2048, 128);
      case 5: return AR_KV_E(4096, 128);
      case 6: return AR_KV_E(8192, 128);
      case 7: return AR_KV_E(16384, 128);
    }
  } else {
    switch (pool.page_log2) {
      case 4: return AR_KV_E(1024, 64);
      case 5: return AR_KV_E(2048, 64);
      case 6: return AR_KV_E(4096, 64);
      case 7: return AR_KV_E(8192, 64);
    }
  }
#undef AR_KV_E
  return cudaErrorInvalidValue;
}

template <bool WRITE>
cudaError_t launch_any(const KvPool& pool, const KvBatch& batch, int dtype, const KvRows& k, const KvRows& v, cudaStream_t stream) {
  const bool f32 = dtype == 0;
  if (pool.e4m3) return f32 ? launch<WRITE, true, true>(pool, batch, k, v, stream) : launch<WRITE, true, false>(pool, batch, k, v, stream);
  return f32 ? launch<WRITE, false, true>(pool, batch, k, v, stream) : launch<WRITE, false, false>(pool, batch, k, v, stream);
}

}  // namespace

cudaError_t launch_kv_append(const KvPool& pool, const KvBatch& batch, int dtype, const KvRows& k, const KvRows& v,
                             cudaStream_t stream) {
  return launch_any<true>(pool, batch, dtype, k, v, stream);
}
cudaError_t launch_kv_read(const KvPool& pool, const KvBatch& batch, int dtype, const KvRows& k, const KvRows& v,
                           cudaStream_t stream) {
  return launch_any<false>(pool, batch, dtype, k, v, stream);
}

}  // namespace ar
