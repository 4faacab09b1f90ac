// Device helpers that the kernels of the 8-bit key/value cache share: which sequence and tile a CTA works on, and what the codes
// stand for.
#pragma once
#include <cuda_fp16.h>

#include "ar_kernels.h"

namespace ar {

// starts[b] held inside [0, T]: the arrays lie in device memory, the host has not seen them.
__device__ __forceinline__ int kv_start(const KvBatch& s, int b) {
  return s.starts ? min(max(s.starts[b], 0), s.T) : b;
}

// A CTA's place in a grid over the tiles of all sequences, whose sizes only the device knows.  A sequence with n rows has
// at most floor(n * rows_per / tile) + slack tiles; so that the first tile of sequence b may stand at
// base(b) = floor(start(b) * rows_per / tile) + slack * b, and floor(T * rows_per / tile) + slack * B places hold them
// all.  The sequence of a place is the last one with base(b) <= place, looked for by a whole warp, 32 candidates at a
// time; a place past its sequence's tiles stays empty.
struct KvPlace {
  int b, tile;     // sequence, tile within it
  int row0, n;     // its rows of the packed tensors
  int length;      // tokens of the sequence, the call's counted in (a negative one counts as 0)
};
__device__ __forceinline__ long long kv_base(const KvBatch& s, int b, int rows_per, int tile_log2, int slack) {
  return (((long long)kv_start(s, b) * rows_per) >> tile_log2) + (long long)slack * b;
}
__device__ __forceinline__ KvPlace kv_place(const KvBatch& s, int place, int rows_per, int tile_log2, int slack) {
  if (!s.starts) {  // one row each: the place says which
    const int tiles = ((rows_per - 1) >> tile_log2) + 1, b = place / tiles;
    return KvPlace{b, place - b * tiles, b, 1, max(s.lengths[b], 0)};
  }
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = s.B;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int b = lo + lane * step;
    const bool le = b < hi && kv_base(s, b, rows_per, tile_log2, slack) <= place;
    const int seen = max(__popc(__ballot_sync(0xffffffffu, le)), 1);
    lo += (seen - 1) * step;
    hi = min(hi, lo + step);
  }
  KvPlace p;
  p.b = lo;
  p.row0 = kv_start(s, lo);
  p.n = max(kv_start(s, lo + 1) - p.row0, 0);
  p.tile = (int)(place - kv_base(s, lo, rows_per, tile_log2, slack));  // (may be negative in front of starts[0])
  p.length = max(s.lengths[lo], 0);
  return p;
}
// Places of such a grid.
inline long long kv_places(const KvBatch& s, int rows_per, int tile_log2, int slack) {
  if (!s.starts) return (((rows_per - 1) >> tile_log2) + 1) * (long long)s.B;
  return (((long long)s.T * rows_per) >> tile_log2) + (long long)slack * s.B;
}

__device__ __forceinline__ void kv_report(const KvBatch& s) {
  if (s.sticky) atomicOr(s.sticky, STATUS_PAGE);
}
// The page that holds block `blk` of sequence b's tokens, or -1 (reported by the caller) where there is none.
__device__ __forceinline__ int kv_page(const KvPool& pool, const KvBatch& s, int b, int blk) {
  if (blk < 0 || blk >= s.table_pages) return -1;
  const int page = s.page_table[(long long)b * s.table_stride + blk];
  return page >= 0 && page < pool.pages ? page : -1;
}

// Programmatic dependent launch: a kernel's launch, and its way to griddepcontrol.wait, which comes before its first access to
// memory, lie under the last CTAs of the kernel before it.
template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
  cudaLaunchAttribute early;
  early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  early.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &early;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

// ---- q ----
// A row of q is taken times 2^-e, its largest element (`top`: the bits of it) then below 2; a logit's factor is 2^e * scale * constant in this order,
// so that neither a subnormal q nor one of 2^127 leaves the range on the way.
__device__ __forceinline__ int kv_binade(uint32_t top) { return min(max((int)(top >> 23) - 127, -126), 127); }
__device__ __forceinline__ float kv_power(int e) {  // -127 <= e <= 127; 2^-127 is subnormal
  return __uint_as_float(e == -127 ? 0x00400000u : (uint32_t)(127 + e) << 23);
}

// ---- references of a softmax ----
// 2^(m + e): m a logit, e a logarithm of a page's scale.  In one number the scale would be lost beside a logit of 2^24 or more, and keys
// whose logits are that large and alike would be weighted by their pages' scales.
struct KvRef {
  float m, e;
};
// log2 of p over q, for a q whose m is not -inf (p's may be).
__device__ __forceinline__ float kv_over(const KvRef& p, const KvRef& q) { return (p.m - q.m) + (p.e - q.e); }
// The larger one; m = -inf: there is none.
__device__ __forceinline__ KvRef kv_larger(const KvRef& p, const KvRef& q) {
  if (p.m == -INFINITY) return q;
  return q.m == -INFINITY || kv_over(p, q) > 0.f ? p : q;
}
// Where a logit may reach this (in the log2 domain), it is added to the page's exponent only after the reference has been taken off it:
// in one f32 number the exponent would be rounded to 2^-5 there.  Ordinary keys and queries stay below (|q| of 64 and keys of 127); the pairs cost the
// few-row kernel 4 to 18 % and the many-row kernel, whose steps have no time to spare, twice the time.
constexpr float KV_LARGE_LOGIT = 64.0f;  // as |q| * scale, codes up to 448 and 128 channels: below 2^20
// 2^e * scale: times sum (q / 2^e) code, below 2^17, and log2(e) / sqrt(D), below 2^-2, a logit is below 2^127.  Beyond it a block's
// logits are NaN, all of them: which ones would be infinite, and of which sign, decides what an infinity is worth.
constexpr float KV_MOST_FACTOR = 5.192296858534828e33f;  // 2^112

// ---- codes ----
// The four codes of w -> f32.
template <bool E4M3>
__device__ __forceinline__ void kv_values4(uint32_t w, float (&x)[4]) {
  if constexpr (E4M3) {
    uint32_t lo, hi;
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
    const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&lo)), q = __half22float2(*reinterpret_cast<const __half2*>(&hi));
    x[0] = p.x; x[1] = p.y; x[2] = q.x; x[3] = q.y;
  } else {  // code + 128 in the low byte of 2^23
    const uint32_t u = w ^ 0x80808080u;
    x[0] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440)) - 8388736.0f;
    x[1] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7441)) - 8388736.0f;
    x[2] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7442)) - 8388736.0f;
    x[3] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7443)) - 8388736.0f;
  }
}
// Two values -> two E4M3 codes, round to nearest even (the caller keeps them inside +-448).
__device__ __forceinline__ uint32_t e4m3_codes(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

}  // namespace ar
