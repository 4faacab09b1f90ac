// Attention over the 8-bit paged cache (include/ar_attn.h, ar_kv_cache_attention).
//
//   logit(r, t) = (q_r . kcode_t) * s_k(page of t) / sqrt(D),   o_r = sum_t p_t * s_v(page of t) * vcode_t / sum_t p_t
//
// Scales are constants of a page, so the products run on the codes themselves.
//   QK   INT8: integer MMAs on the codes as they lie in memory, no conversion; q in fixed point, multiples of 2^-21 of
//        the binade of its row's largest element (a bf16 q exactly, but for elements 2^-14 below it), as three signed 8-bit
//        digits: the sums are exact.  E4M3: codes converted to f16,
//        which holds them exactly; q scaled by a power of two per row to f16 (bf16 exactly, but for elements 2^-14 below the row's
//        largest), f32 tensors as two f16 terms.
//   PV   codes as f16 (exact: 8 and 4 significant bits of 11), P in f16, rounded to nearest; f32 tensors as two f16 terms.
// Accumulators, maxima and sums are 32 bits.
//
// V scales differ by page, and P in f16 must neither overflow nor vanish: with s_v = 2^e * f, 1 <= f < 2, the exponent joins the
// logit: x = logit * log2(e) + e - e_ref, u = 2^(x - m + 12), where m follows the maximum of x (it may lag by up to 2, so
// that accumulators are rescaled rarely) and e_ref is the exponent of the piece's first page; P = u * f < 2^15, and the row
// sum takes u * 2^(e_ref - e).  O is then in units of 2^(m - 12 + e_ref), the sum l in units of 2^(m - 12).
//
// The products are transposed, S^T = K Q^T and O^T = V^T P^T, so that the rows of Q are the narrow side of the MMA (8 columns per
// tile): the query heads of one kv head's group next to one another, then the next token.
//
// What bounds it: memory, 26 bytes of codes per clock and SM.  A 16-token block of D = 128 then has 157 clocks, in which the ALU pipe (64
// lanes per clock) converts V -- 96 instructions for INT8 -- and the MMAs take 32 to 48.  So each warp works by itself:
// groups of 32 keys, a ring of its own in shared memory filled by cp.async, no barrier in the loop; the CTA's four warps
// share a piece of one row tile's keys and join at its end.
#include <cuda_bf16.h>

#include "ar_ptx.cuh"
#include "kv_cache.cuh"

namespace ar {
namespace {
using namespace arptx;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int GROUP = 32;       // keys of a warp's step: two blocks of 16, the smallest page
constexpr int WARPS = 4;
constexpr int SMS = 148;
constexpr int LEAST_UNITS = 4;  // groups of a share: one per warp
constexpr float P_SHIFT = 12.0f, LAG = 2.0f;
constexpr int E_LIMIT = 100;    // largest |e - e_ref|
constexpr float SCALE_FLOOR = 8.673617379884035e-19f;  // 2^-60, the least scale a page is given
constexpr int WHOLE_KEYS = 512;  // up to this length a row tile's keys are not cut

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
__device__ __forceinline__ uint32_t transpose8x8(uint32_t w) {  // of an 8 x 8 matrix of 16-bit elements spread over the warp
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(w));
  return r;
}
// The two codes of the low (HI = 0) or high half of w -> f16x2.  INT8 (w with the sign bits flipped, so the bytes are code +
// 128): the byte under the exponent of 1024 is 1152 + code.
template <bool E4M3, int HI>
__device__ __forceinline__ uint32_t expand2(uint32_t w) {
  if constexpr (E4M3) {
    uint32_t r;
    if constexpr (HI)
      asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(w));
    else
      asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(w));
    return r;
  } else {
    const uint32_t h = __byte_perm(w, 0x64646464u, HI ? 0x4342 : 0x4140);
    const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t unsign(uint32_t w) { return E4M3 ? w : w ^ 0x80808080u; }

// Shared memory keeps the codes in lines of 128 bytes: one token of D = 128, two of D = 64.  The 16-byte piece q of a line
// lies at q ^ swizzle(line), chosen for the reads below: K by rows (8 rows x 4 pieces per phase), V by four tokens
// x 16 or 8 channels per thread (4 token pairs x 2 or 4 pieces per phase); neither has bank conflicts.
template <int D, bool IS_V>
__device__ __forceinline__ int line_swizzle(int line) {
  if (IS_V) return D == 128 ? (line & 6) : (((line & 1) << 2) | (line & 2));
  return D == 128 ? ((line & 1) << 2) : 0;
}
template <int D, bool IS_V>
__device__ __forceinline__ int piece_at(int token, int q) {
  const int line = D == 128 ? token : token >> 1;
  const int c = D == 128 ? q : ((token & 1) << 2) | q;
  return (line << 7) | ((c ^ line_swizzle<D, IS_V>(line)) << 4);
}

template <int D, int NT>
struct Sh {
  static constexpr int ROWS = 8 * NT;
  static constexpr int TILE = GROUP * D;                    // bytes of a group's K or V codes
  static constexpr int CTAS_PER_SM = NT == 1 ? 3 : 2;       // 168 or 255 registers
  static constexpr int STAGES = D == 64 ? 4 : NT == 1 ? 2 : 3;
  static constexpr int RING = STAGES * 2 * TILE;            // per warp
  static constexpr int ML = WARPS * RING;                   // [warp][row]{m, l}
  static constexpr int SCALES = ML + WARPS * ROWS * 8;      // [warp][stage]{s_k, s_v of the first block, s_k, s_v of the second}
  static constexpr int BYTES = SCALES + WARPS * STAGES * 16;
  static_assert(RING >= ROWS * D * 4, "the ring also takes the warp's accumulator at the end of a piece");
  static_assert((BYTES + 1024 + 512) * CTAS_PER_SM <= 228 * 1024, "shared memory of the SM");
};

// What the rows of a sequence see.
struct Seen {
  int total;    // keys of the sequence inside the table and max_length
  int pos0;     // position of the sequence's first row of this call
  int causal;
  __device__ __forceinline__ int limit(int token) const { return causal ? max(min(total, pos0 + token + 1), 0) : total; }
};
__device__ __forceinline__ Seen kv_seen(const KvAttnArgs& a, int length, int n) {
  const long long cap = min((long long)a.batch.table_pages << a.pool.page_log2, (long long)a.max_length);
  Seen s;
  s.total = (int)min((long long)length, cap);
  s.pos0 = length - n;
  s.causal = a.causal;
  return s;
}

// A sequence as the division of the work sees it: `tiles` row tiles per kv head, `groups` groups of keys each (the last row's;
// earlier rows of a causal call see fewer).
struct Work {
  int row0, n, length, tiles, groups;
};
template <int ROWS>
__device__ __forceinline__ Work work_of(const KvAttnArgs& a, int G, int b) {
  Work w;
  w.row0 = kv_start(a.batch, b);
  w.n = a.batch.starts ? max(kv_start(a.batch, b + 1) - w.row0, 0) : 1;
  w.length = max(a.batch.lengths[b], 0);
  w.tiles = (int)(((long long)w.n * G + ROWS - 1) / ROWS);
  w.groups = max(1, (kv_seen(a, w.length, w.n).total + GROUP - 1) / GROUP);
  return w;
}

// Partial results of a cut row tile.  A CTA has two places: 2i for the piece it starts with, which continues the CTA before, and
// 2i + 1 for the piece it ends with, when that begins a cut tile.  A place: ROWS x D values, then per row {m + e_ref, m, l, -}.
template <int D, int ROWS>
__host__ __device__ constexpr int place_floats() { return ROWS * (D + 4); }
// What the join has to know about the cut tile that CTA i begins: packed row of its sequence's first token, first row of
// the tile, rows | kv head << 16, the last CTA with a piece of it (-1: none).
struct Cut {
  int row0, r0;
  uint32_t rows_head;
  int last;
};

template <int D, bool E4M3, bool F32, int NT>
__global__ void __launch_bounds__(WARPS * 32, Sh<D, NT>::CTAS_PER_SM) kv_attn_kernel(const KvAttnArgs a, int whole) {
  using S = Sh<D, NT>;
  constexpr int ROWS = S::ROWS;
  constexpr int QREGS = E4M3 ? (F32 ? 2 : 1) * (D / 16) * 2 : 3 * (D / 32) * 2;
  constexpr int MT = D / 16;  // 16-channel tiles of O^T
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long scan[WARPS];
  __shared__ long long found[2];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * S::RING;
  float* ml = (float*)(smem + S::ML);
  float* scales = (float*)(smem + S::SCALES) + warp * S::STAGES * 4;
  const int G = a.Hq / a.pool.Hkv, Hkv = a.pool.Hkv;

  // ---- this CTA's share: units [u, u_end) of the groups of all row tiles, or one whole row tile ----
  int b = 0;
  long long u = 0, u_end = 0, base = 0;  // base: first unit of sequence b
  int shares = 1;                        // CTAs that have one: share i is [all * i / shares, all * (i + 1) / shares)
  Work w;
  if (whole) {
    const KvPlace p = kv_place(a.batch, blockIdx.x, G, NT == 1 ? 3 : 4, 1);
    if (p.tile < 0 || (long long)p.tile * ROWS >= (long long)p.n * G) return;
    b = p.b;
    w = work_of<ROWS>(a, G, b);
    u = ((long long)blockIdx.y * w.tiles + p.tile) * w.groups;
    u_end = u + w.groups;
  } else {
    const int per = (a.batch.B + WARPS * 32 - 1) / (WARPS * 32);
    const int b0 = threadIdx.x * per, b1 = min(b0 + per, a.batch.B);
    long long mine = 0;
    for (int i = b0; i < b1; i++) {
      const Work x = work_of<ROWS>(a, G, i);
      mine += (long long)x.tiles * x.groups * Hkv;
    }
    long long upto = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane >= s) upto += v;
    }
    if (lane == 31) scan[warp] = upto;
    __syncthreads();
    long long all = 0;
#pragma unroll
    for (int i = 0; i < WARPS; i++) {
      if (i < warp) upto += scan[i];
      all += scan[i];
    }
    shares = (int)max(1ll, min((long long)gridDim.x, all / LEAST_UNITS));
    u = all * blockIdx.x / shares;
    u_end = all * (blockIdx.x + 1) / shares;
    if (blockIdx.x >= shares || all == 0) {
      if (threadIdx.x == 0) ((Cut*)a.partial)[blockIdx.x].last = -1;
      return;
    }
    long long at = upto - mine;
    if (u >= at && u < upto) {
      for (int i = b0; i < b1; i++) {
        const Work x = work_of<ROWS>(a, G, i);
        const long long next = at + (long long)x.tiles * x.groups * Hkv;
        if (u < next) {
          found[0] = i;
          found[1] = at;
          break;
        }
        at = next;
      }
    }
    __syncthreads();
    b = (int)found[0];
    base = found[1];
    w = work_of<ROWS>(a, G, b);
  }
  bool begun_cut = false;

  const int log2 = a.pool.page_log2;
  const long long page_bytes = ((long long)Hkv << log2) * D;
  const int lane_k = (lane >> 3 << 7) | (((lane & 7) ^ line_swizzle<D, false>(lane >> 3)) << 4);
  const int lane_v0 = (lane >> 3 << 7) | (((lane & 7) ^ line_swizzle<D, true>(lane >> 3)) << 4);
  const int lane_v1 = (lane >> 3 << 7) | (((lane & 7) ^ line_swizzle<D, true>((lane >> 3) + 4)) << 4);

  while (true) {  // a piece of one row tile
    const int idx = (int)((u - base) / w.groups), g_begin = (int)(u - base - (long long)idx * w.groups);
    const int g_end = (int)min((long long)w.groups, g_begin + (u_end - u));
    const int h = idx / w.tiles, r0 = (idx - h * w.tiles) * ROWS, rn = min(ROWS, w.n * G - r0);
    const Seen seen = kv_seen(a, w.length, w.n);
    const int end = seen.limit((r0 + rn - 1) / G);    // keys that some row of the tile sees
    const int lim_low = seen.limit(r0 / G);           // that all of them see
    if (seen.total < w.length && g_begin == 0 && threadIdx.x == 0) kv_report(a.batch);
    const int* table = a.batch.page_table + (long long)b * a.batch.table_stride;
    const int stop = min(g_end, (end + GROUP - 1) / GROUP);  // groups past the tile's last key are empty
    const int steps = (stop - g_begin - warp + WARPS - 1) / WARPS;  // (may be negative)

    // ---- the ring: page numbers are read one step ahead ----
    auto page_of = [&](int key) {
      if (key >= end) return -2;  // past the end: nothing to report
      const int pg = table[key >> log2];
      return pg >= 0 && pg < a.pool.pages ? pg : -1;
    };
    int next_page[2];
    auto look = [&](int it) {
      const int key0 = (g_begin + warp + it * WARPS) * GROUP;
      next_page[0] = it < steps ? page_of(key0) : -2;
      next_page[1] = it < steps ? (log2 > 4 ? (key0 + 16 < end ? next_page[0] : -2) : page_of(key0 + 16)) : -2;
    };
    auto fetch = [&](int it) {
      if (it < steps) {
        const int key0 = (g_begin + warp + it * WARPS) * GROUP;
        const uint32_t dst = smem_u32(ring + (it % S::STAGES) * 2 * S::TILE);
        const bool full = key0 + GROUP <= end;
#pragma unroll
        for (int blk = 0; blk < 2; blk++) {
          const int pg = next_page[blk], key = key0 + blk * 16;
          const long long off = (long long)max(pg, 0) * page_bytes + (((long long)h << log2) + (key & ((1 << log2) - 1))) * D + lane * 16;
          const uint8_t *ks = a.pool.k + off, *vs = a.pool.v + off;
          constexpr int COPIES = 16 * D / 512;
          if (full && pg >= 0) {
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
              cp_async16(dst + blk * 16 * D + i * 512 + lane_k, ks + i * 512, true);
              cp_async16(dst + S::TILE + blk * 16 * D + i * 512 + ((i & 1) ? lane_v1 : lane_v0), vs + i * 512, true);
            }
          } else {  // past the last key, or no page: zeros, so that no stale pattern meets a zero weight
            if (pg == -1 && lane == 0) kv_report(a.batch);
#pragma unroll
            for (int i = 0; i < COPIES; i++) {
              const bool in = pg >= 0 && key + (i * 512 + lane * 16) / D < end;
              cp_async16(dst + blk * 16 * D + i * 512 + lane_k, in ? ks + i * 512 : a.pool.k, in);
              cp_async16(dst + S::TILE + blk * 16 * D + i * 512 + ((i & 1) ? lane_v1 : lane_v0), in ? vs + i * 512 : a.pool.v, in);
            }
          }
        }
        if (lane < 4) {
          const int pg = lane & 2 ? next_page[1] : next_page[0];
          float* to = scales + (it % S::STAGES) * 4 + lane;
          if (pg >= 0)
            cp_async4(smem_u32(to), (lane & 1 ? a.pool.v_scale : a.pool.k_scale) + (long long)pg * Hkv + h, true);
          else
            *to = -1.0f;  // no scale is negative: keys to leave out
        }
      }
      cp_async_commit();
    };
    look(0);
#pragma unroll
    for (int it = 0; it < S::STAGES - 1; it++) {
      fetch(it);
      look(it + 1);
    }

    // ---- Q: row g of each tile of 8; word j of a thread's channels starts at channel(j) ----
    auto channel = [&](int j) { return (j >> 2) * 64 + c * 16 + (j & 3) * 4; };
    uint32_t qr[NT][QREGS];
    float row_c[NT][2];  // of rows 2c, 2c + 1: logit in the log2 domain = accumulator * row_c * s_k
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = r0 + nt * 8 + g;
      const bool in = nt * 8 + g < rn;
      const int token = r / G;
      const long long at = (w.row0 + (long long)token) * a.q.st + (long long)(h * G + (r - token * G)) * a.q.sh;
      float v[D / 16][4];
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; j++) {
        if (!in) {
          v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.f;
        } else if constexpr (F32) {
          const float4 x = *(const float4*)((const float*)a.q.p + at + channel(j));
          v[j][0] = x.x; v[j][1] = x.y; v[j][2] = x.z; v[j][3] = x.w;
        } else {
          const uint2 x = *(const uint2*)((const __nv_bfloat16*)a.q.p + at + channel(j));
          v[j][0] = __uint_as_float(x.x << 16);
          v[j][1] = __uint_as_float(x.x & 0xffff0000u);
          v[j][2] = __uint_as_float(x.y << 16);
          v[j][3] = __uint_as_float(x.y & 0xffff0000u);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(v[j][i]));
      }
      bool odd = false;  // NaN or infinity in the row: the integer digits cannot carry it
      if constexpr (!E4M3) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
          for (int i = 0; i < 4; i++) sum += v[j][i] * 0.f;
        odd = sum != 0.f;  // (a NaN: 0 * inf, 0 * NaN)
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^-e brings the largest element below 2; both factors are normal f32 numbers
      const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126);
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      float mine = __uint_as_float((uint32_t)(127 + e) << 23) * ((1.0f / sqrtf((float)D)) * LOG2E);
      if constexpr (E4M3) {
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float x0 = v[j][2 * i] * down, x1 = v[j][2 * i + 1] * down;
            const uint32_t x = pack_half2(x0, x1);
            qr[nt][j * 2 + i] = x;
            if constexpr (F32) qr[nt][(D / 16) * 2 + j * 2 + i] = pack_half2((x0 - half_lo(x)) * 2048.0f, (x1 - half_hi(x)) * 2048.0f);
          }
      } else {
        mine *= 1.0f / 2097152.0f;
        odd = (__ballot_sync(0xffffffffu, odd) >> (lane & 28) & 15u) != 0;
        if (odd) mine = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          uint32_t d0 = 0, d1 = 0, d2 = 0;
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const int x = odd ? 0 : __float2int_rn(v[j][i] * down * 2097152.0f);  // |x| <= 2^22
            const int x1 = (x + 128) >> 8, x2 = (x1 + 128) >> 8;                  // |x2| <= 64
            d0 |= (uint32_t)((x - (x1 << 8)) & 0xff) << (8 * i);
            d1 |= (uint32_t)((x1 - (x2 << 8)) & 0xff) << (8 * i);
            d2 |= (uint32_t)(x2 & 0xff) << (8 * i);
          }
          qr[nt][j] = d0;
          qr[nt][D / 16 + j] = d1;
          qr[nt][D / 8 + j] = d2;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        row_c[nt][i] = __shfl_sync(0xffffffffu, mine, (2 * c + i) * 4);
        const int rr = nt * 8 + 2 * c + i;
        lim[nt][i] = rr < rn ? seen.limit((r0 + rr) / G) : 0;
      }
    }

    // e_ref: the exponent of the piece's first V scale
    auto exponent_of = [](float s) {  // a NaN keeps its NaN in the factor
      const int e = (int)((__float_as_uint(s) >> 23) & 0xffu) - 127;
      return e == 128 ? 0 : max(e, -60);
    };
    int e_ref = 0;
    if (stop > g_begin) {
      const int pg = page_of(g_begin * GROUP);
      if (pg >= 0) e_ref = exponent_of(a.pool.v_scale[(long long)pg * Hkv + h]);
    }

    float o[NT][MT][4];
    float m[NT][2], l[NT][2];  // l: of this thread's keys only, until the end
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < MT; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt][0] = m[nt][1] = -INFINITY;
      l[nt][0] = l[nt][1] = 0.f;
    }

    for (int it = 0; it < steps; it++) {
      fetch(it + S::STAGES - 1);
      look(it + S::STAGES);
      cp_async_wait<S::STAGES - 1>();
      __syncwarp();
      const uint8_t* kt = ring + (it % S::STAGES) * 2 * S::TILE;
      const uint8_t* vt = kt + S::TILE;
      const float4 sc = *(const float4*)(scales + (it % S::STAGES) * 4);
      const int key0 = (g_begin + warp + it * WARPS) * GROUP;

      // S^T = K Q^T: blocks of 16 keys, thread (g, c) has keys g, g + 8 and rows 2c, 2c + 1
      float s[NT][2][4];
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        uint32_t ka[2][D / 16];  // 4 codes each of keys g and g + 8
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
          for (int i = 0; i < D / 64; i++) {
            const uint4 v = *(const uint4*)(kt + piece_at<D, false>(blk * 16 + x * 8 + g, c + i * 4));
            ka[x][i * 4] = v.x; ka[x][i * 4 + 1] = v.y; ka[x][i * 4 + 2] = v.z; ka[x][i * 4 + 3] = v.w;
          }
        if constexpr (E4M3) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++) s[nt][blk][0] = s[nt][blk][1] = s[nt][blk][2] = s[nt][blk][3] = 0.f;
          float t[NT][4];
          if constexpr (F32) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) t[nt][0] = t[nt][1] = t[nt][2] = t[nt][3] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < D / 16; j++) {
            const uint32_t f[4] = {expand2<true, 0>(ka[0][j]), expand2<true, 0>(ka[1][j]), expand2<true, 1>(ka[0][j]), expand2<true, 1>(ka[1][j])};
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
              mma_f16(s[nt][blk], f, qr[nt][j * 2], qr[nt][j * 2 + 1]);
              if constexpr (F32) mma_f16(t[nt], f, qr[nt][(D / 16 + j) * 2], qr[nt][(D / 16 + j) * 2 + 1]);
            }
          }
          if constexpr (F32) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
              for (int i = 0; i < 4; i++) s[nt][blk][i] = fmaf(t[nt][i], 1.0f / 2048.0f, s[nt][blk][i]);
          }
        } else {
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            int t[3][4];
#pragma unroll
            for (int d = 0; d < 3; d++) {
              t[d][0] = t[d][1] = t[d][2] = t[d][3] = 0;
#pragma unroll
              for (int j = 0; j < D / 32; j++)
                mma_s8(t[d], ka[0][2 * j], ka[1][2 * j], ka[0][2 * j + 1], ka[1][2 * j + 1], qr[nt][d * (D / 16) + 2 * j],
                       qr[nt][d * (D / 16) + 2 * j + 1]);
            }
            // each digit's sum is below 2^21: the two low ones fit 32 bits together
#pragma unroll
            for (int i = 0; i < 4; i++) s[nt][blk][i] = fmaf((float)t[2][i], 65536.0f, (float)(t[1][i] * 256 + t[0][i]));
          }
        }
      }

      // scales of the two blocks
      const float sk[2] = {sc.x, sc.z}, sv[2] = {sc.y, sc.w};
      float f[2], w_l[2], ex[2];
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        if (blk == 1 && log2 > 4) {  // one page
          f[1] = f[0]; w_l[1] = w_l[0]; ex[1] = ex[0];
        } else {
          const int e = exponent_of(sv[blk]);
          const float vs = sv[blk] < SCALE_FLOOR ? SCALE_FLOOR : sv[blk];  // (a NaN stays)
          f[blk] = vs * __uint_as_float((uint32_t)(127 - min(e, 126)) << 23) * (e == 127 ? 0.5f : 1.0f);
          const int rel = min(max(e - e_ref, -E_LIMIT), E_LIMIT);
          ex[blk] = (float)rel;
          w_l[blk] = __uint_as_float((uint32_t)(127 - rel) << 23);
        }
      }
      const bool edge = key0 + GROUP > lim_low || sk[0] < 0.f || sk[1] < 0.f;
      float mx[NT][2];
      bool grow = false;
#pragma unroll
      for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
          float top = -INFINITY;
#pragma unroll
          for (int blk = 0; blk < 2; blk++) {
            const float k = row_c[nt][r] * sk[blk];
#pragma unroll
            for (int x = 0; x < 2; x++) {
              float v = fmaf(s[nt][blk][x * 2 + r], k, ex[blk]);
              if (edge && (key0 + blk * 16 + x * 8 + g >= lim[nt][r] || sk[blk] < 0.f)) v = -INFINITY;
              s[nt][blk][x * 2 + r] = v;
              top = fmaxf(top, v);
            }
          }
          mx[nt][r] = top;
          grow = grow || top > m[nt][r] + LAG;
        }
      if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
          for (int r = 0; r < 2; r++) {
            float top = mx[nt][r];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float m_new = fmaxf(m[nt][r], top);
            const float alpha = m[nt][r] == -INFINITY ? 0.f : ex2f(m[nt][r] - m_new);
            m[nt][r] = m_new;
            l[nt][r] *= alpha;
#pragma unroll
            for (int i = 0; i < MT; i++) {
              o[nt][i][r] *= alpha;
              o[nt][i][r + 2] *= alpha;
            }
          }
      }
      uint32_t ph[NT][2][2], pl[F32 ? NT : 1][2][2];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float sum[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
        for (int r = 0; r < 2; r++) {
          const float ref = m[nt][r] == -INFINITY ? 0.f : m[nt][r] - P_SHIFT;
#pragma unroll
          for (int blk = 0; blk < 2; blk++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
              const float p = ex2f(s[nt][blk][x * 2 + r] - ref);
              sum[r][blk] += p;
              s[nt][blk][x * 2 + r] = p * f[blk];
              // a row that does not see the key takes 0 * f: a page's NaN must not reach it
              if (edge && key0 + blk * 16 + x * 8 + g >= lim[nt][r]) s[nt][blk][x * 2 + r] = 0.f;
            }
          l[nt][r] += sum[r][0] * w_l[0] + sum[r][1] * w_l[1];
        }
#pragma unroll
        for (int blk = 0; blk < 2; blk++)
#pragma unroll
          for (int x = 0; x < 2; x++) {
            const float x0 = s[nt][blk][x * 2], x1 = s[nt][blk][x * 2 + 1];
            const uint32_t p = pack_half2(x0, x1);
            ph[nt][blk][x] = transpose8x8(p);
            if constexpr (F32) pl[nt][blk][x] = transpose8x8(pack_half2(x0 - half_lo(p), x1 - half_hi(p)));
          }
      }

      // O^T += V^T P^T, 16 keys per step: tokens 2c, 2c + 1, 2c + 8, 2c + 9, channels 16g .. or 8g ..; tile i has channels 2i, 2i + 1 of those
#pragma unroll
      for (int blk = 0; blk < 2; blk++) {
        uint32_t vw[4][D / 32];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const int t = blk * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
          if constexpr (D == 128) {
            const uint4 x = *(const uint4*)(vt + piece_at<D, true>(t, g));
            vw[i][0] = x.x; vw[i][1] = x.y; vw[i][2] = x.z; vw[i][3] = x.w;
          } else {
            const uint2 x = *(const uint2*)(vt + piece_at<D, true>(t, g >> 1) + (g & 1) * 8);
            vw[i][0] = x.x; vw[i][1] = x.y;
          }
        }
#pragma unroll
        for (int i = 0; i < MT; i++) {
          const uint32_t x0 = unsign<E4M3>(vw[0][i >> 1]), x1 = unsign<E4M3>(vw[1][i >> 1]);
          const uint32_t x2 = unsign<E4M3>(vw[2][i >> 1]), x3 = unsign<E4M3>(vw[3][i >> 1]);
          const uint32_t lo = __byte_perm(x0, x1, i & 1 ? 0x7362 : 0x5140), hi = __byte_perm(x2, x3, i & 1 ? 0x7362 : 0x5140);
          const uint32_t va[4] = {expand2<E4M3, 0>(lo), expand2<E4M3, 1>(lo), expand2<E4M3, 0>(hi), expand2<E4M3, 1>(hi)};
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            if constexpr (F32) mma_f16(o[nt][i], va, pl[nt][blk][0], pl[nt][blk][1]);
            mma_f16(o[nt][i], va, ph[nt][blk][0], ph[nt][blk][1]);
          }
        }
      }
      __syncwarp();  // the stage is read: the next fetch may overwrite it
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- join the warps.  Thread (g, c) has rows 2c, 2c + 1 and D / 8 channels from (D / 8) * g; rows of D floats, the 16-byte piece k of row
    // r at k ^ ((r >> 1) & 3) ----
    float* acc = (float*)ring;
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const int row = nt * 8 + 2 * c + r;
#pragma unroll
        for (int k = 0; k < MT / 2; k++)
          *(float4*)(acc + row * D + (((g * (D / 32) + k) ^ c) << 2)) =
              make_float4(o[nt][2 * k][r], o[nt][2 * k][r + 2], o[nt][2 * k + 1][r], o[nt][2 * k + 1][r + 2]);
        float sum = l[nt][r];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) *(float2*)(ml + (warp * ROWS + row) * 2) = make_float2(m[nt][r], sum);
      }
    __syncthreads();
    const bool first = g_begin == 0, last = g_end == w.groups;
    const bool direct = first && last;
    float* place = nullptr;
    if (!direct) {
      place = a.partial + gridDim.x * (sizeof(Cut) / 4) + (long long)(2 * blockIdx.x + (first ? 1 : 0)) * place_floats<D, ROWS>();
      if (first) {
        begun_cut = true;
        if (threadIdx.x == 0) {
          // the last unit of the tile lies with the CTA whose share holds it
          const long long tail = base + (long long)(idx + 1) * w.groups - 1;
          int cta = blockIdx.x + 1;
          if (u_end <= tail) {
            const long long all = scan[0] + scan[1] + scan[2] + scan[3];
            cta = (int)(tail * shares / all);  // a close guess
            while (all * cta / shares > tail) cta--;
            while (all * (cta + 1) / shares <= tail) cta++;
          }
          ((Cut*)a.partial)[blockIdx.x] = Cut{w.row0, r0, (uint32_t)rn | (uint32_t)h << 16, cta};
        }
      }
    }
    constexpr int PPR = D / 4;  // pieces per row
    for (int i = threadIdx.x; i < rn * PPR; i += WARPS * 32) {
      const int r = i / PPR, piece = i % PPR;
      const int at = r * D + ((piece ^ ((r >> 1) & 3)) << 2);
      float2 x[WARPS];
      float mm = -INFINITY;
#pragma unroll
      for (int v = 0; v < WARPS; v++) {
        x[v] = *(const float2*)(ml + (v * ROWS + r) * 2);
        mm = fmaxf(mm, x[v].x);
      }
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float ll = 0.f;
#pragma unroll
      for (int v = 0; v < WARPS; v++) {
        if (x[v].x == -INFINITY && x[v].y == 0.f) continue;  // (a row of NaN has no maximum but a NaN sum)
        const float scale = x[v].x == mm ? 1.0f : ex2f(x[v].x - mm);
        const float4 y = *(const float4*)((const float*)(smem + v * S::RING) + at);
        sum.x += y.x * scale; sum.y += y.y * scale; sum.z += y.z * scale; sum.w += y.w * scale;
        ll += x[v].y * scale;
      }
      if (direct) {
        const int token = (r0 + r) / G, head = h * G + (r0 + r) - token * G;
        const float inv = ll != 0.f ? __uint_as_float((uint32_t)(127 + e_ref) << 23) / ll : 0.f;
        const long long dst = (w.row0 + (long long)token) * a.o.st + (long long)head * a.o.sh + piece * 4;
        if constexpr (F32)
          *(float4*)((float*)a.o.p + dst) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        else
          *(uint2*)((__nv_bfloat16*)a.o.p + dst) = make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
      } else {
        *(float4*)(place + r * D + piece * 4) = sum;
        if (piece == 0) *(float4*)(place + ROWS * D + r * 4) = make_float4(mm + (float)e_ref, mm, ll, 0.f);
      }
    }

    u += g_end - g_begin;
    if (u >= u_end) break;
    __syncthreads();  // the ring is the next piece's
    if (u - base >= (long long)w.tiles * w.groups * Hkv) {  // the next sequence with rows
      base = u;
      do {
        b++;
        w = work_of<ROWS>(a, G, b);
      } while (w.tiles == 0);
    }
  }
  if (!whole && !begun_cut && threadIdx.x == 0) ((Cut*)a.partial)[blockIdx.x].last = -1;
}

// Joins the pieces of the cut tile that CTA i of the kernel above begins: o = 2^(A - M) sum_p 2^(A_p - A) O_p / sum_p 2^(m_p - M) l_p, with
// A and M the largest of A_p = m_p + e_p and of m_p (log2).  A row is shared by JOIN_WARPS / ROWS warps, the pieces in order.
constexpr int JOIN_WARPS = 16;
template <int D, bool F32, int NT>
__global__ void __launch_bounds__(JOIN_WARPS * 32) kv_join_kernel(const KvAttnArgs a) {
  constexpr int ROWS = 8 * NT, SPLIT = JOIN_WARPS / ROWS, V = D / 32;
  __shared__ float acc[JOIN_WARPS][D];
  __shared__ float sums[JOIN_WARPS];
  const Cut cut = ((const Cut*)a.partial)[blockIdx.x];
  if (cut.last < 0) return;
  const int G = a.Hq / a.pool.Hkv;
  const int rn = (int)(cut.rows_head & 0xffffu), h = (int)(cut.rows_head >> 16);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = warp % ROWS, part = warp / ROWS;
  const int pieces = cut.last - (int)blockIdx.x + 1;
  const float* places = a.partial + gridDim.x * (sizeof(Cut) / 4);
  auto place = [&](int p) {  // the first piece is the owner's second place, the others are first places
    return places + (long long)(p == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + p)) * place_floats<D, ROWS>();
  };
  float A = -INFINITY, M = -INFINITY, l = 0.f;
  float x[V];
#pragma unroll
  for (int d = 0; d < V; d++) x[d] = 0.f;
  if (r < rn) {
    for (int p = lane; p < pieces; p += 32) {
      const float2 e = *(const float2*)(place(p) + ROWS * D + r * 4);
      A = fmaxf(A, e.x);
      M = fmaxf(M, e.y);
    }
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) {
      A = fmaxf(A, __shfl_xor_sync(0xffffffffu, A, s));
      M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
    }
#pragma unroll 4
    for (int p = part; p < pieces; p += SPLIT) {
      const float* src = place(p);
      const float4 e = *(const float4*)(src + ROWS * D + r * 4);
      const bool none = e.y == -INFINITY && e.z == 0.f;
      const float wo = none ? 0.f : ex2f(e.x - A), wl = none ? 0.f : ex2f(e.y - M);
      l += e.z * wl;
      if constexpr (D == 128) {
        const float4 y = *(const float4*)(src + r * D + lane * 4);
        x[0] += y.x * wo; x[1] += y.y * wo; x[2] += y.z * wo; x[3] += y.w * wo;
      } else {
        const float2 y = *(const float2*)(src + r * D + lane * 2);
        x[0] += y.x * wo; x[1] += y.y * wo;
      }
    }
  }
#pragma unroll
  for (int d = 0; d < V; d++) acc[warp][lane * V + d] = x[d];
  if (lane == 0) sums[warp] = l;
  __syncthreads();
  if (part != 0 || r >= rn) return;
#pragma unroll
  for (int s = 1; s < SPLIT; s++) {
    l += sums[r + s * ROWS];
#pragma unroll
    for (int d = 0; d < V; d++) x[d] += acc[r + s * ROWS][lane * V + d];
  }
  const float inv = l != 0.f ? exp2f(A - M) / l : 0.f;
  const int token = (cut.r0 + r) / G, head = h * G + (cut.r0 + r) - token * G;
  const long long dst = (cut.row0 + (long long)token) * a.o.st + (long long)head * a.o.sh + lane * V;
#pragma unroll
  for (int d = 0; d < V; d += 2) {
    if constexpr (F32)
      *(float2*)((float*)a.o.p + dst + d) = make_float2(x[d] * inv, x[d + 1] * inv);
    else
      *(uint32_t*)((__nv_bfloat16*)a.o.p + dst + d) = pack_bf16x2(x[d] * inv, x[d + 1] * inv);
  }
}

template <int D, bool E4M3, bool F32, int NT>
cudaError_t launch(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  using S = Sh<D, NT>;
  auto kern = kv_attn_kernel<D, E4M3, F32, NT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
  if (e != cudaSuccess) return e;
  const dim3 grid = plan.ctas ? dim3((unsigned)plan.ctas)
                              : dim3((unsigned)kv_places(a.batch.B, a.batch.T, a.Hq / a.pool.Hkv, NT == 1 ? 3 : 4, 1), (unsigned)a.pool.Hkv);
  kern<<<grid, WARPS * 32, S::BYTES, stream>>>(a, plan.ctas == 0);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  ++*launches;
  if (plan.ctas) {
    kv_join_kernel<D, F32, NT><<<(unsigned)plan.ctas, JOIN_WARPS * 32, 0, stream>>>(a);
    e = cudaGetLastError();
    if (e == cudaSuccess) ++*launches;
  }
  return e;
}
template <int D, bool E4M3, bool F32>
cudaError_t launch_nt(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  return plan.rows == 8 ? launch<D, E4M3, F32, 1>(a, plan, stream, launches) : launch<D, E4M3, F32, 2>(a, plan, stream, launches);
}

}  // namespace

KvAttnPlan kv_attn_plan(const KvPool& pool, int B, int T, int dtype, int Hq, int max_length, int causal) {
  (void)dtype;
  (void)causal;
  KvAttnPlan p;
  const int G = Hq / pool.Hkv;
  p.rows = (long long)T * G <= 8ll * B ? 8 : 16;
  const long long tiles = kv_places(B, T, G, p.rows == 8 ? 3 : 4, 1) * pool.Hkv;
  p.ctas = SMS * (p.rows == 8 ? Sh<128, 1>::CTAS_PER_SM : Sh<128, 2>::CTAS_PER_SM);
  if (max_length <= WHOLE_KEYS || tiles >= 16 * p.ctas) p.ctas = 0;
  p.workspace = (size_t)p.ctas * (sizeof(Cut) + 2 * sizeof(float) * p.rows * (pool.D + 4));
  return p;
}

cudaError_t launch_kv_attention(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  const bool d128 = a.pool.D == 128, f32 = a.dtype == 0;
  if (a.pool.e4m3) {
    if (d128) return f32 ? launch_nt<128, true, true>(a, plan, stream, launches) : launch_nt<128, true, false>(a, plan, stream, launches);
    return f32 ? launch_nt<64, true, true>(a, plan, stream, launches) : launch_nt<64, true, false>(a, plan, stream, launches);
  }
  if (d128) return f32 ? launch_nt<128, false, true>(a, plan, stream, launches) : launch_nt<128, false, false>(a, plan, stream, launches);
  return f32 ? launch_nt<64, false, true>(a, plan, stream, launches) : launch_nt<64, false, false>(a, plan, stream, launches);
}

}  // namespace ar
