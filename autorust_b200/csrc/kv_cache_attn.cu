// Attention over the 8-bit paged cache (include/ar_attn.h, ar_kv_cache_attention).
//
//   logit(r, t) = (q_r . kcode_t) * s_k(page of t) / sqrt(D),   o_r = sum_t p_t * s_v(page of t) * vcode_t / sum_t p_t
//
// Scales are constants of a page, so the products run on the codes themselves.
//   QK   INT8: integer MMAs on the codes as they lie in memory, no conversion; q in fixed point, multiples of 2^-21 of
//        the binade of its row's largest element (a bf16 q exactly, but for elements 2^-14 below it), as three signed 8-bit
//        digits: the sums are exact.  E4M3: codes converted to f16, which holds them exactly; q scaled by a power of two per
//        row to f16 (bf16 with the same exception), f32 tensors as two f16 terms.
//   PV   codes as f16 (exact: 8 and 4 significant bits of 11), P in f16, rounded to nearest; f32 tensors as two f16 terms.
// Accumulators, maxima and sums are 32 bits.  The tensor cores cut what they add at 2^-24 of the sum, towards zero: over the hundreds of blocks of a long
// sequence that is a bias, up to 1.3e-6 of a result at 12000 keys.  f32 tensors add each block's product of 16 keys to O with rounding additions instead
// (a step of 8 sequences of up to 12219 tokens, 16 kv heads, 12 rows, D = 128: 79 us before, 85 so; with one row no more).
//
// V scales differ by page, and P in f16 must neither overflow nor vanish: with s_v = 2^e * f, 1 <= f < 2, the exponent joins the
// logit: x = logit * log2(e) + e - e_ref, u = 2^(x - m + 12), where m follows the maximum of x (it may lag by up to 2, so
// that accumulators are rescaled rarely) and e_ref is the exponent of the piece's first page, held inside [-5, 20]; P = u * f < 2^15,
// and the row sum takes u * 2^(e_ref - e).  Scales that an append writes are 2^-60 to 2^121: e - e_ref is then -80 to 126, which
// leaves the factor and the sums of 2^31 keys normal f32 numbers.  O is then in units of 2^(m - 12 + e_ref), the sum l in units of 2^(m - 12).
// Beside a page of huge values u may vanish where the row's sum needs it, and beside a large logit e - e_ref is rounded off: from the first V
// scale above 2^20 on, or K scale that with the warp's largest |q| may make a logit of 2^20, a warp's groups keep the reference as a pair (logit, exponent), take
// it off logit and exponent each, and sum 2^(logit - m + 12), exponentials of their own.
//
// Rows go in tiles of 8: the query heads of one kv head's group next to one another, then the next token.  S = Q K^T has the
// digits or terms of 8 rows on the 16-row side of the MMA (two digits of the same rows side by side: one thread gets both
// sums), O^T = V^T P^T has the rows on its 8-column side; S leaves a thread with the very elements of P that the second product
// wants from it.
//
// What bounds it: memory, 26 bytes of codes per clock and SM.  A 16-token block of D = 128 then has 157 clocks, in which the ALU pipe (64
// lanes per clock) converts V -- 96 instructions for INT8 -- and the MMAs take 32 to 48.  So each warp works by itself:
// groups of 32 keys, a ring of its own in shared memory filled by cp.async, no barrier in the loop; the CTA's four warps
// share a piece of one row tile's keys and join at its end.
//
// Measured, one token, 32 query and 8 kv heads, D = 128, kernel and join: 8 sequences of 8192 tokens (INT8, 134 MB) 36.9 us, 131072
// tokens of one (E4M3, 268 MB) 56 us, 4.8 TB/s; from the difference of lengths the loop streams at 6.6 TB/s, and some 15 us of a call are its beginning
// (start, length, page, first codes) and its end (join of the warps, of the pieces).  64 ragged sequences of up to 4096 tokens 67 us.
#include <cuda_bf16.h>

#include "ar_ptx.cuh"
#include "kv_cache.cuh"

#include <algorithm>
#include <type_traits>

namespace ar {
namespace {
using namespace arptx;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int GROUP = 32;       // keys of a warp's step: two blocks of 16, the smallest page
constexpr int WARPS = 4;
constexpr int SMS = 148;
constexpr int LEAST_UNITS = 8;   // of a share
// A row tile counts as its groups and START_UNITS more: beginning a piece (page numbers, Q, the first codes, the join of the
// warps at its end) takes a CTA about as long as that many groups (64 ragged sequences: 75 us with 4, 66 with 9, 67 with 12).
constexpr int START_UNITS = 9;
constexpr float P_SHIFT = 12.0f, LAG = 2.0f;
constexpr float WIDE = 1048576.0f;  // 2^20
constexpr int E_REF_LEAST = -5, E_REF_MOST = 20, E_LIMIT = 126;  // the last: largest e - e_ref
constexpr float SCALE_FLOOR = 8.673617379884035e-19f;  // 2^-60, the least scale a page is given

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// x * 2^d, d <= 0, where 2^d by itself may be below the f32 numbers and x * 2^d is not.
__device__ __forceinline__ float times_ex2(float x, float d) { return x * ex2f(fmaxf(d, -100.0f)) * ex2f(fminf(d + 100.0f, 0.0f)); }
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
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
  static constexpr int ME = ML + WARPS * ROWS * 8;          // [warp][row] the reference's exponent (KvRef::e)
  static constexpr int SCALES = ME + WARPS * ROWS * 4;      // [warp][stage]{s_k, s_v of the first block, s_k, s_v of the second}
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

// Division by a number that the host knows (n < 2^31): by multiplication with its rounded-up reciprocal (Granlund and
// Montgomery, "Division by invariant integers using multiplication").
struct Divider {
  uint32_t m;
  int s1, s2;
  __device__ __forceinline__ int operator()(int n) const {
    const uint32_t t = __umulhi(m, (uint32_t)n);
    return (int)((t + (((uint32_t)n - t) >> s1)) >> s2);
  }
};
Divider divider(uint32_t d) {
  int l = 0;
  while ((1ull << l) < d) l++;
  return Divider{(uint32_t)((((1ull << l) - d) << 32) / d + 1), l < 1 ? l : 1, l > 1 ? l - 1 : 0};
}

// A sequence as the division of the work sees it: `tiles` row tiles per kv head, `groups` groups of keys each (the last row's;
// earlier rows of a causal call see fewer).
struct Work {
  int row0, n, length, tiles, groups;
  __device__ __forceinline__ uint32_t tile_units() const { return (uint32_t)groups + START_UNITS; }
  __device__ __forceinline__ uint32_t units(int Hkv) const { return (uint32_t)tiles * tile_units() * Hkv; }
};
template <int ROWS>
__device__ __forceinline__ void divide(const KvAttnArgs& a, int G, Work& w) {
  w.tiles = (w.n * G + ROWS - 1) / ROWS;
  w.groups = max(1, (kv_seen(a, w.length, w.n).total + GROUP - 1) / GROUP);
}
template <int ROWS>
__device__ __forceinline__ Work work_of(const KvAttnArgs& a, int G, int b) {
  Work w;
  w.row0 = kv_start(a.batch, b);
  w.n = a.batch.starts ? max(kv_start(a.batch, b + 1) - w.row0, 0) : 1;
  w.length = max(a.batch.lengths[b], 0);
  divide<ROWS>(a, G, w);
  return w;
}

// Partial results of a cut row tile.  A CTA has two places: 2i for the piece it starts with, which continues the CTA before, and
// 2i + 1 for the piece it ends with, when that begins a cut tile.  A place: ROWS x D values, then per row {m + e_ref, m, l, 0}, or
// where a warp was far {m, m's exponent, -l, FAR_PIECE + e_ref}: the sign of l (of a zero, too) tells the join, which has no register to spare.
constexpr float FAR_PIECE = 1024.0f;
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
__global__ void __launch_bounds__(WARPS * 32, Sh<D, NT>::CTAS_PER_SM) kv_attn_kernel(const KvAttnArgs a, const Divider by_g, int whole) {
  using S = Sh<D, NT>;
  constexpr int ROWS = S::ROWS;
  // Operands of the QK product, rows 0-7 | 8-15.  E4M3: one row tile, its f16 terms (high | low); two bf16 tiles, one beside the
  // other; two f32 tiles, (high | low) each.  INT8: (digit 2 | digit 1) of each tile, then digit 0 of (tile 0 | tile 1).
  constexpr int QOPS = E4M3 ? (NT == 2 && F32 ? 2 : 1) : NT + 1;
  constexpr int QSTEPS = E4M3 ? D / 16 : D / 32;
  constexpr int MT = D / 16;  // 16-channel tiles of O^T
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * S::RING;
  float* ml = (float*)(smem + S::ML);
  float* me = (float*)(smem + S::ME) + warp * ROWS;
  float* scales = (float*)(smem + S::SCALES) + warp * S::STAGES * 4;
  const int G = a.Hq / a.pool.Hkv, Hkv = a.pool.Hkv;

  asm volatile("griddepcontrol.launch_dependents;");  // what comes next may take its places as CTAs leave; it waits for all of this
  asm volatile("griddepcontrol.wait;" ::: "memory");  // whatever came before in the stream is done and visible

  // ---- this CTA's share: units [u, u_end) of the groups of all row tiles, or one whole row tile ----
  // Every warp works it out for itself, without a barrier; 32-bit numbers, which the host has checked the sizes for.
  int b = 0;
  uint32_t u = 0, u_end = 0, base = 0;     // base: first unit of sequence b
  uint32_t per_share = 1, longer = 0;      // shares of per_share units, the first `longer` ones have one more
  int shares = 1, kv_tile = 0;
  Work w;
  if (whole) {
    const KvPlace p = kv_place(a.batch, blockIdx.x, G, NT == 1 ? 3 : 4, 1);
    if (p.tile < 0 || (long long)p.tile * ROWS >= (long long)p.n * G) return;
    b = p.b;
    kv_tile = p.tile;
    w = Work{p.row0, p.n, p.length, 0, 0};
    divide<ROWS>(a, G, w);
    u = 0;
    u_end = w.tile_units();
  } else {
    const int per = (a.batch.B + 31) / 32;
    const int b0 = lane * per, b1 = min(b0 + per, a.batch.B);
    uint32_t mine = 0;
    Work x{0, 0, 0, 0, 0};
    for (int i = b0; i < b1; i++) {
      x = work_of<ROWS>(a, G, i);
      mine += x.units(Hkv);
    }
    uint32_t upto = mine;
#pragma unroll
    for (int s = 1; s < 32; s <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, s);
      if (lane >= s) upto += v;
    }
    const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
    shares = max(1, (int)min((uint32_t)gridDim.x, all / LEAST_UNITS));
    per_share = all / shares;
    longer = all - per_share * shares;
    u = per_share * blockIdx.x + min(blockIdx.x, longer);
    u_end = u + per_share + (blockIdx.x < longer ? 1u : 0u);
    uint32_t at = upto - mine;
    const uint32_t has = __ballot_sync(0xffffffffu, u >= at && u < upto);
    if (blockIdx.x >= shares || has == 0) {
      if (threadIdx.x == 0) ((Cut*)a.partial)[blockIdx.x].last = -1;
      return;
    }
    const int src = __ffs(has) - 1;
    if (per > 1 && lane == src) {  // which of this lane's sequences
      for (b = b0; b < b1; b++) {
        x = work_of<ROWS>(a, G, b);
        if (u - at < x.units(Hkv)) break;
        at += x.units(Hkv);
      }
    }
    b = __shfl_sync(0xffffffffu, per > 1 ? b : b0, src);
    base = __shfl_sync(0xffffffffu, at, src);
    w.row0 = __shfl_sync(0xffffffffu, x.row0, src);
    w.n = __shfl_sync(0xffffffffu, x.n, src);
    w.length = __shfl_sync(0xffffffffu, x.length, src);
    divide<ROWS>(a, G, w);
  }
  bool begun_cut = false;

  const int log2 = a.pool.page_log2;
  const long long page_bytes = ((long long)Hkv << log2) * D;
  const int lane_k = (lane >> 3 << 7) | (((lane & 7) ^ line_swizzle<D, false>(lane >> 3)) << 4);
  const int lane_v0 = (lane >> 3 << 7) | (((lane & 7) ^ line_swizzle<D, true>(lane >> 3)) << 4);
  const int lane_v1 = (lane >> 3 << 7) | (((lane & 7) ^ line_swizzle<D, true>((lane >> 3) + 4)) << 4);

  while (true) {  // a piece of one row tile
    int h, tile;
    uint32_t from = 0;  // units of the tile in front of this share
    if (whole) {
      h = blockIdx.y;
      tile = kv_tile;
    } else {
      const uint32_t idx = (u - base) / w.tile_units();
      from = u - base - idx * w.tile_units();
      h = (int)(idx / (uint32_t)w.tiles);
      tile = (int)(idx - h * w.tiles);
    }
    const uint32_t to = min(w.tile_units(), from + (u_end - u));
    const int g_begin = max((int)from - START_UNITS, 0), g_end = (int)to - START_UNITS;
    if (g_end <= 0) break;  // the share ends before the tile's first group: the next one begins the tile
    const int r0 = tile * ROWS, rn = min(ROWS, w.n * G - r0);
    const Seen seen = kv_seen(a, w.length, w.n);
    const int end = seen.limit(by_g(r0 + rn - 1));    // keys that some row of the tile sees
    const int lim_low = seen.limit(by_g(r0));           // that all of them see
    if (seen.total < w.length && g_begin == 0 && threadIdx.x == 0) kv_report(a.batch);
    const int* table = a.batch.page_table + (long long)b * a.batch.table_stride;
    const int stop = min(g_end, (end + GROUP - 1) / GROUP);  // groups past the tile's last key are empty
    const int steps = (stop - g_begin - warp + WARPS - 1) / WARPS;  // (may be negative)

    // ---- Q is asked for before the codes, which would keep it waiting: row g of each tile of 8; word j of a thread's channels
    // starts at channel(j) ----
    auto channel = [&](int j) { return (j >> 2) * 64 + c * 16 + (j & 3) * 4; };
    float qv[NT][D / 16][4];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      const int r = r0 + nt * 8 + g;
      const int token = by_g(r);
      const long long at = (w.row0 + (long long)token) * a.q.st + (long long)(h * G + (r - token * G)) * a.q.sh;
#pragma unroll
      for (int j = 0; j < D / 16; j++) {
        float(&v)[4] = qv[nt][j];
        if (nt * 8 + g >= rn) {
          v[0] = v[1] = v[2] = v[3] = 0.f;
        } else if constexpr (F32) {
          const float4 x = *(const float4*)((const float*)a.q.p + at + channel(j));
          v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        } else {
          const uint2 x = *(const uint2*)((const __nv_bfloat16*)a.q.p + at + channel(j));
          v[0] = __uint_as_float(x.x << 16);
          v[1] = __uint_as_float(x.x & 0xffff0000u);
          v[2] = __uint_as_float(x.y << 16);
          v[3] = __uint_as_float(x.y & 0xffff0000u);
        }
      }
    }

    // ---- the ring: page numbers are read one step ahead ----
    auto page_of = [&](int key) {
      if (key >= end) return -2;  // past the end: nothing to report
      const int pg = table[key >> log2];
      return pg >= 0 && pg < a.pool.pages ? pg : -1;
    };
    // e_ref: the exponent of the piece's first V scale, but inside limits
    auto exponent_of = [](float s) {  // a NaN keeps its NaN in the factor
      const int e = (int)((__float_as_uint(s) >> 23) & 0xffu) - 127;
      return e == 128 ? 0 : max(e, -60);
    };
    int e_ref = 0;
    const int page0 = page_of(g_begin * GROUP);
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
    if (page0 >= 0) e_ref = min(max(exponent_of(a.pool.v_scale[(long long)page0 * Hkv + h]), E_REF_LEAST), E_REF_MOST);
#pragma unroll
    for (int it = 0; it < S::STAGES - 1; it++) {
      fetch(it);
      look(it + 1);
    }

    uint32_t q_top = 0;  // of the warp's rows
    uint32_t qa[QOPS][QSTEPS][4] = {};
    float row_c[NT];  // of row g: logit in the log2 domain = accumulator * (row_c * s_k * unit)
    const float unit = (1.0f / sqrtf((float)D)) * LOG2E * (E4M3 ? 1.0f : 1.0f / 2097152.0f);
    int lim[NT];      // keys that row g sees
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
      float(&v)[D / 16][4] = qv[nt];
      lim[nt] = nt * 8 + g < rn ? seen.limit(by_g(r0 + nt * 8 + g)) : 0;
      uint32_t top = 0;  // bits of the largest |q|; infinities and NaN are the largest patterns
#pragma unroll
      for (int j = 0; j < D / 16; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = max(top, __float_as_uint(v[j][i]) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (top < 0x7f800000u) q_top = max(q_top, top);
      const int e = kv_binade(top);
      const float down = kv_power(-e);
      row_c[nt] = kv_power(e);
      const bool odd = top >= 0x7f800000u;  // the row is NaN
      if (odd) row_c[nt] = __uint_as_float(0x7fc00000u);
      if constexpr (E4M3) {
#pragma unroll
        for (int j = 0; j < D / 16; j++)
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float x0 = v[j][2 * i] * down, x1 = v[j][2 * i + 1] * down;
            const uint32_t x = pack_half2(x0, x1);
            if constexpr (F32) {
              qa[nt][j][2 * i] = x;
              qa[nt][j][2 * i + 1] = pack_half2((x0 - half_lo(x)) * 2048.0f, (x1 - half_hi(x)) * 2048.0f);
            } else {
              qa[0][j][2 * i + nt] = x;
            }
          }
      } else {
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
          int x0[4], x1[4], x2[4];  // |x0| <= 2^22 and its signed digits: the low bytes of x0, x1 and x2, |x2| <= 64
#pragma unroll
          for (int i = 0; i < 4; i++) {
            x0[i] = odd ? 0 : __float2int_rn(v[j][i] * down * 2097152.0f);
            x1[i] = (x0[i] + 128) >> 8;
            x2[i] = (x1[i] + 128) >> 8;
          }
          auto low_bytes = [](const int (&x)[4]) { return __byte_perm(__byte_perm(x[0], x[1], 0x0040), __byte_perm(x[2], x[3], 0x0040), 0x5410); };
          const uint32_t d0 = low_bytes(x0), d1 = low_bytes(x1), d2 = low_bytes(x2);
          qa[nt][j >> 1][(j & 1) * 2] = d2;
          qa[nt][j >> 1][(j & 1) * 2 + 1] = d1;
          qa[NT][j >> 1][(j & 1) * 2 + nt] = d0;
        }
      }
    }

    float o[NT][MT][4];
    float m[NT], l[NT];  // of row g; l: of this thread's keys only, until the end
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int i = 0; i < MT; i++) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      m[nt] = -INFINITY;
      l[nt] = 0.f;
    }

    // From the first V scale above WIDE, or K scale above sk_most, on: scales and logits may be far apart.
    bool far = false;
    const float sk_most = KV_LARGE_LOGIT * kv_power(-kv_binade(__reduce_max_sync(0xffffffffu, q_top)));
    if (lane < ROWS) me[lane] = 0.f;

    // One group of keys.  EDGE: some row does not see all of them, or there are keys to leave out, or far.
    auto step = [&](auto edge_c, int it) {
      constexpr bool EDGE = decltype(edge_c)::value;
      const bool pairs = EDGE && far;
      const uint8_t* kt = ring + (it % S::STAGES) * 2 * S::TILE;
      const uint8_t* vt = kt + S::TILE;
      const float4 sc = *(const float4*)(scales + (it % S::STAGES) * 4);
      const int key0 = (g_begin + warp + it * WARPS) * GROUP;

      // S = Q K^T: tiles of 8 keys, thread (g, c) has row g and keys 2c, 2c + 1
      float s[NT][4][2];
#pragma unroll
      for (int n8 = 0; n8 < 4; n8++) {
        uint32_t kw[D / 16];  // 4 codes each of key g
#pragma unroll
        for (int i = 0; i < D / 64; i++) {
          const uint4 v = *(const uint4*)(kt + piece_at<D, false>(n8 * 8 + g, c + i * 4));
          kw[i * 4] = v.x; kw[i * 4 + 1] = v.y; kw[i * 4 + 2] = v.z; kw[i * 4 + 3] = v.w;
        }
        if constexpr (E4M3) {
          float t[QOPS][4] = {};
#pragma unroll
          for (int j = 0; j < QSTEPS; j++) {
            const uint32_t b0 = expand2<true, 0>(kw[j]), b1 = expand2<true, 1>(kw[j]);
#pragma unroll
            for (int i = 0; i < QOPS; i++) mma_f16(t[i], qa[i][j], b0, b1);
          }
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
              if constexpr (F32)
                s[nt][n8][i] = fmaf(t[nt][2 + i], 1.0f / 2048.0f, t[nt][i]);
              else
                s[nt][n8][i] = t[0][2 * nt + i];
            }
        } else {
          int t[QOPS][4] = {};
#pragma unroll
          for (int j = 0; j < QSTEPS; j++)
#pragma unroll
            for (int i = 0; i < QOPS; i++) mma_s8(t[i], qa[i][j], kw[2 * j], kw[2 * j + 1]);
          // each digit's sum is at most 2^21: the two low ones fit 32 bits together
#pragma unroll
          for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int i = 0; i < 2; i++) s[nt][n8][i] = fmaf((float)t[nt][i], 65536.0f, (float)(t[nt][2 + i] * 256 + t[NT][2 * nt + i]));
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
          const int rel = min(e - e_ref, E_LIMIT);
          ex[blk] = (float)rel;
          w_l[blk] = __uint_as_float((uint32_t)(127 - rel) << 23);
        }
      }
      auto rescale = [&](int nt, float alpha) {  // the accumulators of this thread are rows 2c and 2c + 1
        const float al[2] = {__shfl_sync(0xffffffffu, alpha, 8 * c), __shfl_sync(0xffffffffu, alpha, 8 * c + 4)};
#pragma unroll
        for (int i = 0; i < MT; i++)
#pragma unroll
          for (int x = 0; x < 4; x++) o[nt][i][x] *= al[x & 1];
      };
      if (pairs) {  // s becomes the logit alone, the reference a pair
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          KvRef most{-INFINITY, 0.f};
#pragma unroll
          for (int blk = 0; blk < 2; blk++) {
            float k = row_c[nt] * sk[blk];
            k = k > KV_MOST_FACTOR ? __uint_as_float(0x7fc00000u) : k * unit;
            float top = -INFINITY;
#pragma unroll
            for (int n8 = 2 * blk; n8 < 2 * blk + 2; n8++)
#pragma unroll
              for (int i = 0; i < 2; i++) {
                float v = __fmul_rn(s[nt][n8][i], k);
                if (key0 + n8 * 8 + 2 * c + i >= lim[nt] || sk[blk] < 0.f) v = -INFINITY;
                s[nt][n8][i] = v;
                top = fmaxf(top, v);
              }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            most = kv_larger(KvRef{top, ex[blk]}, most);
          }
          const KvRef ref{m[nt], me[nt * 8 + g]};
          float alpha = 1.0f;
          if (most.m != -INFINITY && (ref.m == -INFINITY || kv_over(most, ref) > LAG)) {
            const float d = ref.m == -INFINITY ? -INFINITY : kv_over(ref, most);
            alpha = ex2f(d);
            l[nt] = times_ex2(l[nt], d);
            m[nt] = most.m;
          }
          __syncwarp();
          if (c == 0 && alpha != 1.0f) me[nt * 8 + g] = most.e;
          __syncwarp();
          if (__any_sync(0xffffffffu, alpha != 1.0f)) rescale(nt, alpha);
        }
      } else {
        float mx[NT];
        bool grow = false;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
          float top = -INFINITY;
#pragma unroll
          for (int n8 = 0; n8 < 4; n8++) {
            const float k = row_c[nt] * sk[n8 >> 1] * unit;
#pragma unroll
            for (int i = 0; i < 2; i++) {
              float v = fmaf(s[nt][n8][i], k, ex[n8 >> 1]);
              if (EDGE && (key0 + n8 * 8 + 2 * c + i >= lim[nt] || sk[n8 >> 1] < 0.f)) v = -INFINITY;
              s[nt][n8][i] = v;
              top = fmaxf(top, v);
            }
          }
          mx[nt] = top;
          grow = grow || top > m[nt] + LAG;
        }
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int nt = 0; nt < NT; nt++) {
            float top = mx[nt];
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const float m_new = fmaxf(m[nt], top);
            const float alpha = m[nt] == -INFINITY ? 0.f : ex2f(m[nt] - m_new);
            l[nt] = m[nt] == -INFINITY ? l[nt] * 0.f : EDGE ? times_ex2(l[nt], m[nt] - m_new) : l[nt] * alpha;
            m[nt] = m_new;
            rescale(nt, alpha);
          }
        }
      }
      uint32_t ph[NT][4];
      [[maybe_unused]] uint32_t pl[F32 ? NT : 1][4];
#pragma unroll
      for (int nt = 0; nt < NT; nt++) {
        float sum[2] = {0.f, 0.f};
        const float ref = m[nt] == -INFINITY ? 0.f : pairs ? m[nt] : m[nt] - P_SHIFT;
        const float me_row = pairs ? me[nt * 8 + g] - P_SHIFT : 0.f;
#pragma unroll
        for (int n8 = 0; n8 < 4; n8++) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float x = s[nt][n8][i] - ref;
            const float p = ex2f(pairs ? x + (ex[n8 >> 1] - me_row) : x);
            sum[n8 >> 1] += pairs ? ex2f(x - me_row) : p;
            s[nt][n8][i] = p * f[n8 >> 1];
            // a row that does not see the key takes 0 * f: a page's NaN must not reach it
            if (EDGE && key0 + n8 * 8 + 2 * c + i >= lim[nt]) s[nt][n8][i] = 0.f;
          }
          const float x0 = s[nt][n8][0], x1 = s[nt][n8][1];
          ph[nt][n8] = pack_half2(x0, x1);
          if constexpr (F32) pl[nt][n8] = pack_half2(x0 - half_lo(ph[nt][n8]), x1 - half_hi(ph[nt][n8]));
        }
        l[nt] += pairs ? sum[0] + sum[1] : sum[0] * w_l[0] + sum[1] * w_l[1];
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
            if constexpr (F32) {
              float part[4] = {0.f, 0.f, 0.f, 0.f};
              mma_f16(part, va, pl[nt][2 * blk], pl[nt][2 * blk + 1]);
              mma_f16(part, va, ph[nt][2 * blk], ph[nt][2 * blk + 1]);
#pragma unroll
              for (int x = 0; x < 4; x += 2)
                unpack_f32x2(add_f32x2(pack_f32x2(o[nt][i][x], o[nt][i][x + 1]), pack_f32x2(part[x], part[x + 1])), o[nt][i][x], o[nt][i][x + 1]);
            } else {
              mma_f16(o[nt][i], va, ph[nt][2 * blk], ph[nt][2 * blk + 1]);
            }
          }
        }
      }
    };

    for (int it = 0; it < steps; it++) {
      fetch(it + S::STAGES - 1);
      look(it + S::STAGES);
      cp_async_wait<S::STAGES - 1>();
      __syncwarp();
      const float4 sc = *(const float4*)(scales + (it % S::STAGES) * 4);
      if (fmaxf(sc.y, sc.w) > WIDE || fmaxf(sc.x, sc.z) > sk_most) far = true;
      const bool edge = (g_begin + warp + it * WARPS) * GROUP + GROUP > lim_low || fminf(sc.x, sc.z) < 0.f || far;
      if (__builtin_expect(edge, 0))
        step(std::true_type{}, it);
      else
        step(std::false_type{}, it);
      __syncwarp();  // the stage is read: the next fetch may overwrite it
    }
    cp_async_wait<0>();
    __syncwarp();

    // ---- join the warps.  Thread (g, c) has rows 2c, 2c + 1 and D / 8 channels from (D / 8) * g; rows of D floats, the 16-byte piece k of row
    // r at k ^ ((r >> 1) & 3) ----
    float* acc = (float*)ring;
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
#pragma unroll
      for (int r = 0; r < 2; r++) {
        const int row = nt * 8 + 2 * c + r;
#pragma unroll
        for (int k = 0; k < MT / 2; k++)
          *(float4*)(acc + row * D + (((g * (D / 32) + k) ^ c) << 2)) =
              make_float4(o[nt][2 * k][r], o[nt][2 * k][r + 2], o[nt][2 * k + 1][r], o[nt][2 * k + 1][r + 2]);
      }
      float sum = l[nt];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (c == 0) *(float2*)(ml + (warp * ROWS + nt * 8 + g) * 2) = make_float2(m[nt], sum);
    }
    const bool some_far = __syncthreads_or(far);
    const bool first = g_begin == 0, last = g_end == w.groups;
    const bool direct = first && last;
    float* place = nullptr;
    if (!direct) {
      place = a.partial + gridDim.x * (sizeof(Cut) / 4) + (long long)(2 * blockIdx.x + (first ? 1 : 0)) * place_floats<D, ROWS>();
      if (first) {
        begun_cut = true;
        if (threadIdx.x == 0) {
          // the last unit of the tile lies with the CTA whose share holds it
          const uint32_t tail = u - from + w.tile_units() - 1, split = (per_share + 1) * longer;
          const uint32_t cta = tail < split ? tail / (per_share + 1) : longer + (tail - split) / per_share;
          ((Cut*)a.partial)[blockIdx.x] = Cut{w.row0, r0, (uint32_t)rn | (uint32_t)h << 16, (int)min(cta, (uint32_t)shares - 1)};
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
      const float base = mm == -INFINITY ? 0.f : mm;
      float ref = 0.f;  // the row's reference is 2^(base + ref)
      if (some_far) {
        ref = -INFINITY;
#pragma unroll
        for (int v = 0; v < WARPS; v++) {
          x[v].x = (x[v].x - base) + ((const float*)(smem + S::ME))[v * ROWS + r];
          ref = fmaxf(ref, x[v].x);
        }
        if (ref == -INFINITY) ref = 0.f;
      }
      float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
      float ll = 0.f;
#pragma unroll
      for (int v = 0; v < WARPS; v++) {
        if (x[v].x == -INFINITY && x[v].y == 0.f) continue;  // (a row of NaN has no maximum but a NaN sum)
        const float d = some_far ? x[v].x - ref : x[v].x - base;
        const float scale = ex2f(d);
        const float4 y = *(const float4*)((const float*)(smem + v * S::RING) + at);
        sum.x += y.x * scale; sum.y += y.y * scale; sum.z += y.z * scale; sum.w += y.w * scale;
        ll += times_ex2(x[v].y, d);
      }
      if (direct) {
        const int token = by_g(r0 + r), head = h * G + (r0 + r) - token * G;
        const float inv = ll != 0.f ? __uint_as_float((uint32_t)(127 + e_ref) << 23) / ll : 0.f;
        const long long dst = (w.row0 + (long long)token) * a.o.st + (long long)head * a.o.sh + piece * 4;
        if constexpr (F32)
          *(float4*)((float*)a.o.p + dst) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
        else
          *(uint2*)((__nv_bfloat16*)a.o.p + dst) = make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
      } else {
        *(float4*)(place + r * D + piece * 4) = sum;
        if (piece == 0) *(float4*)(place + ROWS * D + r * 4) = some_far ? make_float4(mm, ref, -ll, (float)e_ref + FAR_PIECE) : make_float4(mm + (float)e_ref, mm, ll, 0.f);
      }
    }

    u += to - from;
    if (u >= u_end) break;
    __syncthreads();  // the ring is the next piece's
    if (u - base >= w.units(Hkv)) {  // the next sequence with rows
      base = u;
      w.tiles = 0;
      while (w.tiles == 0 && ++b < a.batch.B) w = work_of<ROWS>(a, G, b);
      if (b >= a.batch.B) break;  // (starts that overlap: more rows than there are)
    }
  }
  if (!whole && !begun_cut && threadIdx.x == 0) ((Cut*)a.partial)[blockIdx.x].last = -1;
}

// Joins the pieces of the cut tiles: o = 2^(A - M) sum_p 2^(A_p - A) O_p / sum_p 2^(m_p - M) l_p, with A and M the largest of
// A_p = m_p + e_p and of m_p (log2).  CTA (x, y) takes the tiles that the CTAs x, x + gridDim.x, .. of the kernel above begin, and of
// those the rows y, y + 4, ..; its warps share a row's pieces, each against maxima of its own, and the row's first warp joins
// them, always in the same order.  A few small CTAs: they are in place and waiting before the last CTA above has left.
constexpr int JOIN_WARPS = 8, JOIN_STEP = 7, JOIN_Y = 4;

// A lane's values of a row, to `dst` in the tensor.
template <int D, bool F32>
__device__ __forceinline__ void store_row(void* dst, const float (&x)[D / 32], float inv) {
#pragma unroll
  for (int d = 0; d < D / 32; d += 2) {
    if constexpr (F32)
      *(float2*)((float*)dst + d) = make_float2(x[d] * inv, x[d + 1] * inv);
    else
      *(uint32_t*)((__nv_bfloat16*)dst + d) = pack_bf16x2(x[d] * inv, x[d + 1] * inv);
  }
}
// Row r of a tile with far pieces, by one warp, references as distances from the largest logit among them.  (A function of its own: such
// pieces are rare, and the others' loop has no registers to spare.)
template <int D, bool F32, int ROWS>
__device__ __noinline__ void join_far(const float* places, int first, int pieces, int r, void* dst) {
  constexpr int V = D / 32;
  auto place = [&](int p) { return places + (long long)(p == 0 ? 2 * first + 1 : 2 * (first + p)) * place_floats<D, ROWS>(); };
  auto row = [&](int p) {  // {m, m's exponent, l, e_ref}
    const float4 e = *(const float4*)(place(p) + ROWS * D + r * 4);
    return e.w == 0.f ? make_float4(e.y, 0.f, e.z, e.y == -INFINITY ? 0.f : e.x - e.y) : make_float4(e.x, e.y, -e.z, e.w - FAR_PIECE);
  };
  float top = -INFINITY, A = -INFINITY, M = -INFINITY, l = 0.f;
  for (int p = 0; p < pieces; p++) top = fmaxf(top, row(p).x);
  const float base = top == -INFINITY ? 0.f : top;
  for (int p = 0; p < pieces; p++) {
    const float4 e = row(p);
    M = fmaxf(M, (e.x - base) + e.y);
    A = fmaxf(A, (e.x - base) + (e.y + e.w));
  }
  float x[V];
#pragma unroll
  for (int d = 0; d < V; d++) x[d] = 0.f;
  for (int p = 0; p < pieces; p++) {
    const float4 e = row(p);
    const bool none = e.x == -INFINITY;  // zeros, or in a row of NaN a NaN sum: 0 * NaN is wanted
    const float wo = none ? 0.f : ex2f((e.x - base) + (e.y + e.w) - A);
    l += times_ex2(e.z, none ? -INFINITY : (e.x - base) + e.y - M);
#pragma unroll
    for (int d = 0; d < V; d++) x[d] += place(p)[r * D + (threadIdx.x & 31) * V + d] * wo;
  }
  store_row<D, F32>(dst, x, l != 0.f ? exp2f(A - M) / l : 0.f);
}

template <int D, bool F32, int NT>
__global__ void __launch_bounds__(JOIN_WARPS * 32, 3) kv_join_kernel(const KvAttnArgs a, const Divider by_g, int ctas) {
  constexpr int ROWS = 8 * NT, V = D / 32;
  __shared__ float acc[JOIN_WARPS][D];
  __shared__ float4 sums[JOIN_WARPS];  // A, M, l, the signs
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // all of the kernel above has left and is visible
  const int G = a.Hq / a.pool.Hkv;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float* places = a.partial + ctas * (sizeof(Cut) / 4);
  for (int first = blockIdx.x; first < ctas; first += gridDim.x) {
    const Cut cut = ((const Cut*)a.partial)[first];
    const int rn = (int)(cut.rows_head & 0xffffu), h = (int)(cut.rows_head >> 16);
    if (cut.last < 0 || (int)blockIdx.y >= rn) continue;
    const int mine = (rn - (int)blockIdx.y + JOIN_Y - 1) / JOIN_Y;  // rows of this CTA, at most 4
    const int width = mine > 2 ? 4 : mine;                          // warps side by side
    const int k = warp % width, part = warp / width, split = JOIN_WARPS / width;
    const int r = (int)blockIdx.y + k * JOIN_Y;
    const int pieces = cut.last - first + 1;
    float A = -INFINITY, M = -INFINITY, l = 0.f;
    uint32_t signs = 0;  // of the pieces' l
    float x[V];
#pragma unroll
    for (int d = 0; d < V; d++) x[d] = 0.f;
    if (r < rn) {
      for (int p0 = part; p0 < pieces; p0 += split * JOIN_STEP) {
        float4 e[JOIN_STEP];
        float y[JOIN_STEP][V];
#pragma unroll
        for (int i = 0; i < JOIN_STEP; i++) {
          const int p = p0 + i * split;
          e[i] = make_float4(-INFINITY, -INFINITY, 0.f, 0.f);
#pragma unroll
          for (int d = 0; d < V; d++) y[i][d] = 0.f;
          if (p < pieces) {  // the first piece is the owner's second place, the others are first places
            const float* src = places + (long long)(p == 0 ? 2 * first + 1 : 2 * (first + p)) * place_floats<D, ROWS>();
            e[i] = *(const float4*)(src + ROWS * D + r * 4);
            signs |= __float_as_uint(e[i].z);
            if constexpr (D == 128) {
              const float4 v = *(const float4*)(src + r * D + lane * 4);
              y[i][0] = v.x; y[i][1] = v.y; y[i][2] = v.z; y[i][3] = v.w;
            } else {
              const float2 v = *(const float2*)(src + r * D + lane * 2);
              y[i][0] = v.x; y[i][1] = v.y;
            }
          }
        }
        float A_new = A, M_new = M;
#pragma unroll
        for (int i = 0; i < JOIN_STEP; i++) {
          A_new = fmaxf(A_new, e[i].x);
          M_new = fmaxf(M_new, e[i].y);
        }
        const float old_o = A == -INFINITY ? 0.f : ex2f(A - A_new), old_d = M == -INFINITY ? -INFINITY : M - M_new;
        l = times_ex2(l, old_d);  // (0 * NaN is wanted: a row of NaN has no maximum)
#pragma unroll
        for (int d = 0; d < V; d++) x[d] *= old_o;
        A = A_new;
        M = M_new;
#pragma unroll
        for (int i = 0; i < JOIN_STEP; i++) {
          const bool none = e[i].y == -INFINITY && e[i].z == 0.f;
          const float wo = none || A == -INFINITY ? 0.f : ex2f(e[i].x - A), wd = none || M == -INFINITY ? -INFINITY : e[i].y - M;
          l += times_ex2(e[i].z, wd);
#pragma unroll
          for (int d = 0; d < V; d++) x[d] += y[i][d] * wo;
        }
      }
    }
    __syncthreads();  // (the tile before has been read)
#pragma unroll
    for (int d = 0; d < V; d++) acc[warp][lane * V + d] = x[d];
    if (lane == 0) sums[warp] = make_float4(A, M, l, __uint_as_float(signs));
    __syncthreads();
    if (part != 0 || r >= rn) continue;
    for (int i = 1; i < split; i++) {
      A = fmaxf(A, sums[k + i * width].x);
      M = fmaxf(M, sums[k + i * width].y);
      signs |= __float_as_uint(sums[k + i * width].w);
    }
    l = 0.f;
#pragma unroll
    for (int d = 0; d < V; d++) x[d] = 0.f;
    for (int i = 0; i < split; i++) {
      const float4 e = sums[k + i * width];
      const float wo = e.x == -INFINITY ? 0.f : ex2f(e.x - A), wd = e.y == -INFINITY ? -INFINITY : e.y - M;
      l += times_ex2(e.z, wd);
#pragma unroll
      for (int d = 0; d < V; d++) x[d] += acc[k + i * width][lane * V + d] * wo;
    }
    const int token = by_g(cut.r0 + r), head = h * G + (cut.r0 + r) - token * G;
    const long long at = (cut.row0 + (long long)token) * a.o.st + (long long)head * a.o.sh + lane * V;
    void* dst = (char*)a.o.p + at * (F32 ? 4 : 2);
    if (signs >> 31)
      join_far<D, F32, ROWS>(places, first, pieces, r, dst);
    else
      store_row<D, F32>(dst, x, l != 0.f ? exp2f(A - M) / l : 0.f);
  }
}

template <int D, bool E4M3, bool F32, int NT>
cudaError_t launch(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  using S = Sh<D, NT>;
  auto kern = kv_attn_kernel<D, E4M3, F32, NT>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::BYTES);
  if (e != cudaSuccess) return e;
  const dim3 grid = plan.ctas ? dim3((unsigned)plan.ctas)
                              : dim3((unsigned)kv_places(a.batch, a.Hq / a.pool.Hkv, NT == 1 ? 3 : 4, 1), (unsigned)a.pool.Hkv);
  const Divider by_g = divider((uint32_t)(a.Hq / a.pool.Hkv));
  e = launch_early(kern, grid, dim3(WARPS * 32), S::BYTES, stream, a, by_g, plan.ctas == 0 ? 1 : 0);
  if (e != cudaSuccess) return e;
  ++*launches;
  if (plan.ctas) {
    e = launch_early(kv_join_kernel<D, F32, NT>, dim3(SMS, JOIN_Y), dim3(JOIN_WARPS * 32), 0, stream, a, by_g, plan.ctas);
    if (e == cudaSuccess) ++*launches;
  }
  return e;
}
template <int D, bool E4M3, bool F32>
cudaError_t launch_nt(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  return plan.rows == 8 ? launch<D, E4M3, F32, 1>(a, plan, stream, launches) : launch<D, E4M3, F32, 2>(a, plan, stream, launches);
}

}  // namespace

// The kernels' times in microseconds, estimated from the call's sizes, decide between this one and the tensor cores' and on the
// latter's parts.  Fitted to measured calls (1 to 64 sequences, 4 to 1024 rows x 1 to 16 heads, 64 to 16384 keys): this
// kernel takes 1.45 ns (D = 64: 1.1) per row tile and group of keys over the whole GPU, the other a 128-key step of 256 rows in
// 2.3 us (1.9) on one SM and 6 us for a CTA's beginning and end; partial results pass memory twice.  8 rows x 4 heads of one
// sequence against 4096 keys: 17 us here, 72 there; 64 rows of 16 sequences against 2048: 231 and 62; 128 rows of 4
// sequences against 16384: 749 here, 324 there in one part, 189 in four.
KvAttnPlan kv_attn_plan(const KvPool& pool, const KvBatch& batch, int dtype, int Hq, int max_length, int causal) {
  (void)causal;
  KvAttnPlan p;
  const int G = Hq / pool.Hkv;
  const long long mean_rows = ((long long)batch.T * G + batch.B - 1) / batch.B;
  p.rows = mean_rows <= 8 ? 8 : 16;
  p.parts = 1;
  if (dtype != 0 && mean_rows > 16) {
    const double per_group = pool.D == 128 ? 1.45e-3 : 1.1e-3, per_step = pool.D == 128 ? 2.3 : 1.9;
    const double pairs = (double)batch.B * pool.Hkv;
    const double here = (max_length <= 512 ? 6.0 : 14.0) +
                        pairs * ((mean_rows + 15) / 16) * ((max_length + GROUP - 1) / GROUP + START_UNITS) * per_group;
    const long long steps = (max_length + 127) / 128, ctas = batch.B * (long long)pool.Hkv * ((mean_rows + 255) / 256);
    auto bytes = [&](long long parts) { return parts > 1 ? sizeof(float) * (size_t)parts * batch.T * Hq * (pool.D + 4) : 0; };
    auto there = [&](long long parts) {
      return 5.0 + (double)((ctas * parts + SMS - 1) / SMS) * (6.0 + per_step * (double)((steps + parts - 1) / parts)) +
             (parts > 1 ? 6.0 + 2.0 * (double)bytes(parts) / 4e6 : 0.0);
    };
    long long parts = std::max(1ll, std::min(std::min((long long)SMS / ctas, 16ll), steps / 4));
    if (there(1) < there(parts)) parts = 1;
    if (there(parts) < here) {
      p.rows = 256;
      p.ctas = 0;
      p.parts = (int)parts;
      p.workspace = bytes(parts);
      return p;
    }
  }
  const long long tiles = batch.B * (long long)pool.Hkv * ((mean_rows + p.rows - 1) / p.rows), groups = (max_length + GROUP - 1) / GROUP;
  const long long most_tiles = kv_places(batch, G, p.rows == 8 ? 3 : 4, 1) * pool.Hkv;
  p.ctas = SMS * (p.rows == 8 ? Sh<128, 1>::CTAS_PER_SM : Sh<128, 2>::CTAS_PER_SM);
  // Cut or whole, again by estimated times: a step of a whole tile's four warps takes 1.05 us (D = 64: 0.85; f32 tensors and
  // 16 rows a quarter more), the codes pass at 4.6 TB/s; shares pass them at 6.0 and cost 10.5 us and 35 ns a tile for
  // being found and joined.  One sequence, 32 / 8 heads, D = 128: 7.7 us whole and 10.7 cut at 512 keys, 36 and 12.6 at
  // 4096; 32 sequences: 20 and 28 at 1024, 58 and 60 at 4096.
  const double step = (pool.D == 128 ? 1.05 : 0.85) * (dtype == 0 ? 1.25 : 1.0) * (p.rows == 8 ? 1.0 : 1.25);
  const double megabytes = 2.0 * pool.D * GROUP * (double)groups * (double)tiles / 1e6;
  const double whole = 4.0 + std::max((double)((tiles + p.ctas - 1) / p.ctas) * (double)((groups + WARPS - 1) / WARPS) * step, megabytes / 4.6 + 3.0);
  const double cut = 10.5 + megabytes / 6.0 + 0.035 * (double)tiles;
  if (whole <= cut || most_tiles * (groups + START_UNITS) > 0xffffffffll) p.ctas = 0;  // (units are 32-bit numbers)
  p.workspace = (size_t)p.ctas * (sizeof(Cut) + 2 * sizeof(float) * p.rows * (pool.D + 4));
  return p;
}

cudaError_t launch_kv_attention(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  const bool d128 = a.pool.D == 128, f32 = a.dtype == 0;
  if (plan.rows == 256) return launch_kv_attention_tc(a, plan.parts, stream, launches);
  if (a.pool.e4m3) {
    if (d128) return f32 ? launch_nt<128, true, true>(a, plan, stream, launches) : launch_nt<128, true, false>(a, plan, stream, launches);
    return f32 ? launch_nt<64, true, true>(a, plan, stream, launches) : launch_nt<64, true, false>(a, plan, stream, launches);
  }
  if (d128) return f32 ? launch_nt<128, false, true>(a, plan, stream, launches) : launch_nt<128, false, false>(a, plan, stream, launches);
  return f32 ? launch_nt<64, false, true>(a, plan, stream, launches) : launch_nt<64, false, false>(a, plan, stream, launches);
}

}  // namespace ar
