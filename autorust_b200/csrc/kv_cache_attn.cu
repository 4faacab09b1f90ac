// Attention over the 8-bit paged cache (include/ar_attn.h, ar_kv_cache_attention).
//
//   logit(r, t) = (q_r . kcode_t) * s_k(page of t) / sqrt(D),   o_r = sum_t p_t * s_v(page of t) * vcode_t / sum_t p_t
//
// Scales are constants of a page, so the products run on the codes themselves, which f16 holds exactly (INT8: 8 bits of its
// 11; E4M3: 4): S = Q Kcode^T and O = P' Vcode by mma.m16n8k16 with f32 accumulation.  The rounding that is left is that of the
// f16 operands Q and P': q is scaled by a power of two per row (a bf16 q is then exact but for elements 2^-14 below the row's
// largest), and f32 tensors keep both as two f16 terms, 22 bits.
//
// V scales differ by page, and P' in f16 must neither overflow nor vanish: with s_v = 2^e * f, 1 <= f < 2, the exponent joins the
// logit: x = logit * log2(e) + e - e_ref, u = 2^(x - m + 12), where m is the running maximum of x and e_ref the exponent of the
// first page of the chunk; P' = u * f <= 2^13, and the row sum takes u * 2^(e_ref - e).  O is then in units of
// 2^(m - 12 + e_ref), the sum l in units of 2^(m - 12).
//
// One CTA: 16 rows of one kv head (the query heads of a token's group next to one another, then the next token) against
// one chunk of the keys.  Its four warps take groups of 32 keys in turn, each with a ring of its own in shared memory that
// cp.async fills (no barrier in the loop), and join their running maxima, sums and accumulators at the end; rows whose keys are
// cut into several chunks leave partial results that a second kernel joins, chunk by chunk in order.
#include <cuda_bf16.h>

#include "ar_ptx.cuh"
#include "kv_cache.cuh"

namespace ar {
namespace {
using namespace arptx;

constexpr float LOG2E = 1.4426950408889634f;
constexpr int M_ROWS = 16;      // rows of a CTA
constexpr int GROUP = 32;       // keys of a warp's step: two blocks of 16, the smallest page
constexpr int WARPS = 4;
constexpr int STAGES = 3;
constexpr float P_SHIFT = 12.0f;
constexpr int E_LIMIT = 100;    // largest |e - e_ref|

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float half_lo(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w & 0xffffu))); }
__device__ __forceinline__ float half_hi(uint32_t w) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }

// Two codes in bytes SEL0 and SEL1 of w -> f16x2.  INT8 (w with the sign bits flipped, so the bytes are code + 128): the byte
// under the exponent of 1024 is 1152 + code.  E4M3: see e4m3_value; the result is 2^-8 of the value.
template <bool E4M3, int SEL0, int SEL1>
__device__ __forceinline__ uint32_t expand2(uint32_t w) {
  if constexpr (E4M3) {
    const uint32_t h = __byte_perm(w, 0u, 0x0404 | (SEL0 << 4) | (SEL1 << 12));
    return (h & 0x80008000u) | ((h >> 1) & 0x3f803f80u);
  } else {
    const uint32_t h = __byte_perm(w, 0x64646464u, 0x4040 | SEL0 | (SEL1 << 8));
    __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&h), __half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480)));
    return *reinterpret_cast<uint32_t*>(&v);
  }
}
template <bool E4M3>
__device__ __forceinline__ uint32_t unsign(uint32_t w) { return E4M3 ? w : w ^ 0x80808080u; }

// Shared memory keeps the codes in lines of 128 bytes: one token of D = 128, two of D = 64.  The 16-byte piece q of a line
// lies at q ^ swizzle(line), chosen for the reads below: K by rows (8 rows x 4 pieces per phase), V by four tokens
// x 16 or 8 channels per thread (4 token pairs x 2 or 4 pieces per phase); neither has bank conflicts.
template <int D, bool IS_V>
__device__ __forceinline__ int piece_at(int token, int q) {
  const int line = D == 128 ? token : token >> 1;
  const int c = D == 128 ? q : ((token & 1) << 2) | q;
  int x;
  if (IS_V)
    x = D == 128 ? (token & 6) : (((line & 1) << 2) | (line & 2));
  else
    x = D == 128 ? ((token & 1) << 2) : 0;
  return (line << 7) | ((c ^ x) << 4);
}

template <int D>
struct Sh {
  static constexpr int TILE = GROUP * D;                    // bytes of a group's K or V codes
  static constexpr int RING = STAGES * 2 * TILE;            // per warp
  static constexpr int SCALES = STAGES * 4;                 // floats per warp: s_k and s_v of the stage's two blocks
  static constexpr int BYTES = WARPS * (RING + SCALES * 4) + WARPS * M_ROWS * 8;
  static_assert(RING >= M_ROWS * D * 4, "the ring also takes the warp's accumulator at the end");
};

// What the rows of a tile see: keys [0, end) of the sequence, row r of the tile up to limit(r).
struct Seen {
  int total;    // keys of the sequence inside the table and max_length
  int pos0;     // position of the sequence's first row of this call
  int causal;
  __device__ __forceinline__ int limit(int token) const { return causal ? max(min(total, pos0 + token + 1), 0) : total; }
};
__device__ __forceinline__ Seen kv_seen(const KvAttnArgs& a, const KvPlace& p) {
  const long long cap = min((long long)a.batch.table_pages << a.pool.page_log2, (long long)a.max_length);
  Seen s;
  s.total = (int)min((long long)p.length, cap);
  s.pos0 = p.length - p.n;
  s.causal = a.causal;
  return s;
}
// Chunks of a tile whose last token is `last`.
__device__ __forceinline__ int kv_chunks(const Seen& s, int last, int chunk) { return max(1, (s.limit(last) + chunk - 1) / chunk); }

// One row of partial results: D accumulated values, then m + e_ref, m, l.
template <int D>
__device__ __forceinline__ float* partial_row(float* base, long long rows, int chunk, long long row) {
  return base + ((long long)chunk * rows + row) * (D + 4);
}

template <int D, bool E4M3, bool F32>
__global__ void __launch_bounds__(WARPS * 32, 2)
kv_attn_kernel(const KvAttnArgs a, int chunk) {
  using S = Sh<D>;
  constexpr int KSTEPS = D / 16;
  extern __shared__ __align__(128) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * S::RING;
  float* scales = (float*)(smem + WARPS * S::RING) + warp * S::SCALES;
  float* ml = (float*)(smem + WARPS * (S::RING + S::SCALES * 4));  // [warp][row]{m, l}

  const int G = a.Hq / a.pool.Hkv;
  const KvPlace p = kv_place(a.batch, blockIdx.x, G, 4, 1);
  const int rows = p.n * G;
  if (p.tile < 0 || p.tile * M_ROWS >= rows) return;
  const int r0 = p.tile * M_ROWS, rn = min(M_ROWS, rows - r0);
  const Seen seen = kv_seen(a, p);
  const int end = seen.limit((r0 + rn - 1) / G);
  const int nchunks = kv_chunks(seen, (r0 + rn - 1) / G, chunk);
  const int ci = blockIdx.z;
  if (ci >= nchunks) return;
  if (seen.total < p.length && ci == 0 && threadIdx.x == 0) kv_report(a.batch);
  const int h = blockIdx.y;
  const int k_begin = ci * chunk, k_end = min(end, k_begin + chunk);
  const int groups = k_end > k_begin ? (k_end - k_begin + GROUP - 1) / GROUP : 0;
  const int log2 = a.pool.page_log2;
  const int* table = a.batch.page_table + (long long)p.b * a.batch.table_stride;

  // ---- the ring ----
  auto fetch = [&](int it) {  // the warp's it-th group
    const int grp = warp + it * WARPS;
    if (grp < groups) {
      const int key0 = k_begin + grp * GROUP;
      int page[2];
#pragma unroll
      for (int b = 0; b < 2; b++) {
        const int key = key0 + b * 16;
        page[b] = -1;
        if (key < k_end) {
          page[b] = table[key >> log2];
          if (page[b] < 0 || page[b] >= a.pool.pages) {
            page[b] = -1;
            if (lane == 0) kv_report(a.batch);
          }
        }
      }
      const uint32_t dst = smem_u32(ring + (it % STAGES) * 2 * S::TILE);
      constexpr int PIECES = D / 16;            // 16-byte pieces of a token
      constexpr int PER = GROUP * PIECES / 32;  // per lane
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const int idx = i * 32 + lane, t = idx / PIECES, q = idx % PIECES;
        const int pg = page[t >> 4];
        const bool in = pg >= 0 && key0 + t < k_end;
        const long long off = in ? ((((long long)pg * a.pool.Hkv + h) << log2) + ((key0 + t) & ((1 << log2) - 1))) * D + q * 16 : 0;
        cp_async16(dst + piece_at<D, false>(t, q), a.pool.k + off, in);
        cp_async16(dst + S::TILE + piece_at<D, true>(t, q), a.pool.v + off, in);
      }
      if (lane < 4) {
        const int pg = page[lane >> 1];
        const float* src = (lane & 1 ? a.pool.v_scale : a.pool.k_scale) + (pg >= 0 ? (long long)pg * a.pool.Hkv + h : 0);
        cp_async4(smem_u32(scales + (it % STAGES) * 4 + lane), src, pg >= 0);  // (zero where there is no page)
      }
    }
    cp_async_commit();
  };
#pragma unroll
  for (int it = 0; it < STAGES - 1; it++) fetch(it);

  // ---- Q: rows g and g + 8 of the tile; channel 16 * (piece) + 4 * j + {0..3} is columns {2c, 2c+1, 2c+8, 2c+9} of step j ----
  uint32_t qh[KSTEPS][4], ql[F32 ? KSTEPS : 1][4];
  float row_c[2];  // logit in the log2 domain = accumulator * row_c * s_k
  int lim[2];
#pragma unroll
  for (int half = 0; half < 2; half++) {
    const int r = r0 + g + half * 8;
    const bool in = r < r0 + rn;
    const int token = r / G;
    lim[half] = in ? seen.limit(token) : 0;
    const long long at = (p.row0 + (long long)token) * a.q.st + (long long)(h * G + (r - token * G)) * a.q.sh;
    float v[KSTEPS][4];
    float top = 0.f;
#pragma unroll
    for (int j = 0; j < KSTEPS; j++) {
      const int d = (j >> 2) * 64 + c * 16 + (j & 3) * 4;
      if (!in) {
        v[j][0] = v[j][1] = v[j][2] = v[j][3] = 0.f;
      } else if constexpr (F32) {
        const float4 w = *(const float4*)((const float*)a.q.p + at + d);
        v[j][0] = w.x; v[j][1] = w.y; v[j][2] = w.z; v[j][3] = w.w;
      } else {
        const uint2 w = *(const uint2*)((const __nv_bfloat16*)a.q.p + at + d);
        v[j][0] = __uint_as_float(w.x << 16);
        v[j][1] = __uint_as_float(w.x & 0xffff0000u);
        v[j][2] = __uint_as_float(w.y << 16);
        v[j][3] = __uint_as_float(w.y & 0xffff0000u);
      }
#pragma unroll
      for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(v[j][i]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // 2^-e brings the largest element below 2; both factors are normal f32 numbers
    const int e = min(max((int)(__float_as_uint(top) >> 23) - 127, -100), 126);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    row_c[half] = __uint_as_float((uint32_t)(127 + e) << 23) * ((1.0f / sqrtf((float)D)) * LOG2E * (E4M3 ? 256.0f : 1.0f));
#pragma unroll
    for (int j = 0; j < KSTEPS; j++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float x0 = v[j][2 * i] * down, x1 = v[j][2 * i + 1] * down;
        const uint32_t w = pack_half2(x0, x1);
        qh[j][half + 2 * i] = w;
        if constexpr (F32) ql[j][half + 2 * i] = pack_half2((x0 - half_lo(w)) * 2048.0f, (x1 - half_hi(w)) * 2048.0f);
      }
    }
  }

  // e_ref: the exponent of the chunk's first V scale
  auto exponent_of = [](float s) {  // of a scale at least 2^-60; a NaN keeps its NaN in the factor
    const int e = (int)((__float_as_uint(s) >> 23) & 0xffu) - 127;
    return e == 128 ? 0 : max(e, -60);
  };
  int e_ref = 0;
  if (groups > 0) {
    const int pg = table[k_begin >> log2];
    if (pg >= 0 && pg < a.pool.pages) e_ref = exponent_of(a.pool.v_scale[(long long)pg * a.pool.Hkv + h]);
  }

  float o[D / 8][4];
#pragma unroll
  for (int i = 0; i < D / 8; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};  // l: this thread's columns only, until the end
  const int lim_low = seen.limit(r0 / G);                   // the least of the tile's rows

  for (int it = 0; warp + it * WARPS < groups; it++) {
    fetch(it + STAGES - 1);
    cp_async_wait<STAGES - 1>();
    __syncwarp();
    const uint8_t* kt = ring + (it % STAGES) * 2 * S::TILE;
    const uint8_t* vt = kt + S::TILE;
    const float4 sc = *(const float4*)(scales + (it % STAGES) * 4);
    const int key0 = k_begin + (warp + it * WARPS) * GROUP;

    // S = Q K^T, 4 blocks of 8 keys
    float s[4][4];
#pragma unroll
    for (int nf = 0; nf < 4; nf++) {
      s[nf][0] = s[nf][1] = s[nf][2] = s[nf][3] = 0.f;
      uint32_t kw[D / 16];  // 4 codes each, steps j = 0 ..
#pragma unroll
      for (int i = 0; i < D / 64; i++) {
        const uint4 w = *(const uint4*)(kt + piece_at<D, false>(nf * 8 + g, c + i * 4));
        kw[i * 4] = w.x; kw[i * 4 + 1] = w.y; kw[i * 4 + 2] = w.z; kw[i * 4 + 3] = w.w;
      }
      uint32_t kb[KSTEPS][2];
#pragma unroll
      for (int j = 0; j < KSTEPS; j++) {
        const uint32_t w = unsign<E4M3>(kw[j]);
        kb[j][0] = expand2<E4M3, 0, 1>(w);
        kb[j][1] = expand2<E4M3, 2, 3>(w);
      }
      if constexpr (F32) {
#pragma unroll
        for (int j = 0; j < KSTEPS; j++) mma16816(s[nf], ql[j], kb[j][0], kb[j][1]);
#pragma unroll
        for (int i = 0; i < 4; i++) s[nf][i] *= 1.0f / 2048.0f;
      }
#pragma unroll
      for (int j = 0; j < KSTEPS; j++) mma16816(s[nf], qh[j], kb[j][0], kb[j][1]);
    }

    // scales of the two blocks
    const float sk[2] = {sc.x, sc.z}, sv[2] = {sc.y, sc.w};
    float f[2], w_l[2], ex[2];
#pragma unroll
    for (int b = 0; b < 2; b++) {
      const int e = exponent_of(sv[b]);
      const float vs = sv[b] < 8.673617379884035e-19f ? 8.673617379884035e-19f : sv[b];  // (a NaN stays)
      f[b] = vs * __uint_as_float((uint32_t)(127 - min(e, 126)) << 23) * (e == 127 ? 0.5f : 1.0f);
      const int rel = min(max(e - e_ref, -E_LIMIT), E_LIMIT);
      ex[b] = (float)rel;
      w_l[b] = __uint_as_float((uint32_t)(127 - rel) << 23);
    }
    const bool edge = key0 + GROUP > lim_low;
    bool hole[2] = {false, false};  // blocks without a page
    {
      const bool whole = key0 + 16 < k_end;
      const int pg0 = table[key0 >> log2], pg1 = whole ? table[(key0 + 16) >> log2] : 0;
      hole[0] = pg0 < 0 || pg0 >= a.pool.pages;
      hole[1] = pg1 < 0 || pg1 >= a.pool.pages;
    }
#pragma unroll
    for (int half = 0; half < 2; half++) {
      float mx = -INFINITY;
#pragma unroll
      for (int nf = 0; nf < 4; nf++) {
        const float k = row_c[half] * sk[nf >> 1];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float x = fmaf(s[nf][half * 2 + i], k, ex[nf >> 1]);
          if (edge || hole[nf >> 1]) {
            const int key = key0 + nf * 8 + c * 2 + i;
            if (key >= lim[half] || hole[nf >> 1]) x = -INFINITY;
          }
          s[nf][half * 2 + i] = x;
          mx = fmaxf(mx, x);
        }
      }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float m_new = fmaxf(m[half], mx);
      const float ref = m_new == -INFINITY ? 0.f : m_new - P_SHIFT;
      const float alpha = m[half] == -INFINITY ? 0.f : ex2f(m[half] - m_new);
      m[half] = m_new;
      float sum[2] = {0.f, 0.f};
#pragma unroll
      for (int nf = 0; nf < 4; nf++) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const float u = ex2f(s[nf][half * 2 + i] - ref);
          sum[nf >> 1] += u;
          s[nf][half * 2 + i] = u * f[nf >> 1];
        }
      }
      l[half] = l[half] * alpha + sum[0] * w_l[0] + sum[1] * w_l[1];
#pragma unroll
      for (int i = 0; i < D / 8; i++) {
        o[i][half * 2] *= alpha;
        o[i][half * 2 + 1] *= alpha;
      }
    }
    // a row that does not see a block at all takes 0 * f there: f of a page poisoned by NaN must not reach it
#pragma unroll
    for (int nf = 0; nf < 4; nf++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (edge && key0 + nf * 8 + c * 2 + (i & 1) >= lim[i >> 1]) s[nf][i] = 0.f;

    // O += P' V, 16 keys per step; token pairs (2c, 2c+1) and (2c+8, 2c+9) of channels 16g.. or 8g..
#pragma unroll
    for (int b = 0; b < 2; b++) {
      uint32_t ph[4], pl[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float x0 = s[2 * b + (i >> 1)][(i & 1) * 2], x1 = s[2 * b + (i >> 1)][(i & 1) * 2 + 1];
        ph[i] = pack_half2(x0, x1);
        if constexpr (F32) pl[i] = pack_half2(x0 - half_lo(ph[i]), x1 - half_hi(ph[i]));
      }
      uint32_t vw[4][D / 32];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int t = b * 16 + 2 * c + (i & 1) + (i >> 1) * 8;
        if constexpr (D == 128) {
          const uint4 w = *(const uint4*)(vt + piece_at<D, true>(t, g));
          vw[i][0] = w.x; vw[i][1] = w.y; vw[i][2] = w.z; vw[i][3] = w.w;
        } else {
          const uint2 w = *(const uint2*)(vt + piece_at<D, true>(t, g >> 1) + (g & 1) * 8);
          vw[i][0] = w.x; vw[i][1] = w.y;
        }
      }
#pragma unroll
      for (int w = 0; w < D / 32; w++) {
        const uint32_t x0 = unsign<E4M3>(vw[0][w]), x1 = unsign<E4M3>(vw[1][w]), x2 = unsign<E4M3>(vw[2][w]), x3 = unsign<E4M3>(vw[3][w]);
#pragma unroll
        for (int hf = 0; hf < 2; hf++) {  // channels 4w + 2hf, 4w + 2hf + 1
          const uint32_t lo = __byte_perm(x0, x1, hf ? 0x7362 : 0x5140), hi = __byte_perm(x2, x3, hf ? 0x7362 : 0x5140);
          const uint32_t a0 = expand2<E4M3, 0, 1>(lo), a1 = expand2<E4M3, 0, 1>(hi);
          const uint32_t b0 = expand2<E4M3, 2, 3>(lo), b1 = expand2<E4M3, 2, 3>(hi);
          float(&oa)[4] = o[w * 4 + hf * 2];
          float(&ob)[4] = o[w * 4 + hf * 2 + 1];
          if constexpr (F32) {
            mma16816(oa, pl, a0, a1);
            mma16816(ob, pl, b0, b1);
          }
          mma16816(oa, ph, a0, a1);
          mma16816(ob, ph, b0, b1);
        }
      }
    }
    __syncwarp();  // the stage is read: the next fetch may overwrite it
  }
  cp_async_wait<0>();
  __syncwarp();

  // ---- join the warps ----
#pragma unroll
  for (int half = 0; half < 2; half++) {
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
    l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
    if (c == 0) {
      ml[(warp * M_ROWS + g + half * 8) * 2] = m[half];
      ml[(warp * M_ROWS + g + half * 8) * 2 + 1] = l[half];
    }
  }
  // Accumulators: thread (g, c) holds channels 2c * (D / 8) .. + D / 4 of its rows, element i of the first half in o[i], of the second
  // in the odd columns.  Rows of D floats; the 16-byte piece k of a thread's run lies at k ^ (lane & 7).
  float* acc = (float*)ring;
  constexpr int RUN = D / 16;  // pieces of a thread's run
#pragma unroll
  for (int half = 0; half < 2; half++) {
#pragma unroll
    for (int k = 0; k < RUN; k++) {
      const int col = k / (RUN / 2), i = (k % (RUN / 2)) * 4;
      const float4 w = make_float4(o[i][half * 2 + col], o[i + 1][half * 2 + col], o[i + 2][half * 2 + col], o[i + 3][half * 2 + col]);
      *(float4*)(acc + (g + half * 8) * D + c * (D / 4) + ((k ^ (lane & (RUN - 1))) << 2)) = w;
    }
  }
  __syncthreads();
  const bool direct = nchunks == 1;
  const long long all_rows = (long long)a.batch.T * a.Hq;
  constexpr int PPR = D / 4;  // pieces per row
  for (int idx = threadIdx.x; idx < rn * PPR; idx += WARPS * 32) {
    const int r = idx / PPR, piece = idx % PPR;
    const int oc = piece / RUN, ok = piece % RUN;  // owner column group and piece of its run
    const int at = r * D + oc * (D / 4) + ((ok ^ (((r & 7) * 4 + oc) & (RUN - 1))) << 2);
    float mm = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; w++) mm = fmaxf(mm, ml[(w * M_ROWS + r) * 2]);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    float ll = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; w++) {
      const float mw = ml[(w * M_ROWS + r) * 2];
      if (mw == -INFINITY && ml[(w * M_ROWS + r) * 2 + 1] == 0.f) continue;  // (a NaN row has no maximum but a NaN sum)
      const float scale = mw == mm ? 1.0f : ex2f(mw - mm);
      const float4 x = *(const float4*)((const float*)(smem + w * S::RING) + at);
      sum.x += x.x * scale; sum.y += x.y * scale; sum.z += x.z * scale; sum.w += x.w * scale;
      ll += ml[(w * M_ROWS + r) * 2 + 1] * scale;
    }
    const int token = (r0 + r) / G, head = h * G + (r0 + r) - token * G;
    if (direct) {
      const float inv = ll != 0.f ? __uint_as_float((uint32_t)(127 + e_ref) << 23) / ll * (E4M3 ? 256.0f : 1.0f) : 0.f;
      const long long dst = (p.row0 + (long long)token) * a.o.st + (long long)head * a.o.sh + piece * 4;
      if constexpr (F32)
        *(float4*)((float*)a.o.p + dst) = make_float4(sum.x * inv, sum.y * inv, sum.z * inv, sum.w * inv);
      else
        *(uint2*)((__nv_bfloat16*)a.o.p + dst) = make_uint2(pack_bf16x2(sum.x * inv, sum.y * inv), pack_bf16x2(sum.z * inv, sum.w * inv));
    } else {
      float* dst = partial_row<D>(a.partial, all_rows, ci, (p.row0 + (long long)token) * a.Hq + head);
      *(float4*)(dst + piece * 4) = sum;
      if (piece == 0) *(float4*)(dst + D) = make_float4(mm + (float)e_ref, mm, ll, 0.f);
    }
  }
}

// Joins the chunks of a row: o = sum_i 2^(A_i - A) O_i * 2^(A - M) / sum_i 2^(m_i - M) l_i, with A and M the largest of A_i = m_i + e_i and
// of m_i (both in log2).  One warp per row.
template <int D, bool E4M3, bool F32>
__global__ void __launch_bounds__(128)
kv_join_kernel(const KvAttnArgs a, int chunk) {
  const int lane = threadIdx.x & 31;
  const long long wid = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const long long all_rows = (long long)a.batch.T * a.Hq;
  if (wid >= all_rows) return;
  const int row = (int)(wid / a.Hq), head = (int)(wid - (long long)row * a.Hq);
  const int G = a.Hq / a.pool.Hkv;
  const KvPlace p = kv_place(a.batch, row, 1, 0, 0);  // tiles of one row: the sequence that holds it
  const int i = row - p.row0;
  if (i < 0 || i >= p.n) return;  // a row of no sequence
  const Seen seen = kv_seen(a, p);
  const int tile_end = min(((i * G + head % G) / M_ROWS + 1) * M_ROWS, p.n * G) - 1;
  const int n = kv_chunks(seen, tile_end / G, chunk);
  if (n == 1) return;  // written by its only chunk
  float A = -INFINITY, M = -INFINITY;
  for (int k = lane; k < n; k += 32) {
    const float2 e = *(const float2*)(partial_row<D>(a.partial, all_rows, k, wid) + D);
    A = fmaxf(A, e.x);
    M = fmaxf(M, e.y);
  }
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    A = fmaxf(A, __shfl_xor_sync(0xffffffffu, A, s));
    M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, s));
  }
  float acc[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; d++) acc[d] = 0.f;
  float l = 0.f;
#pragma unroll 4
  for (int k = 0; k < n; k++) {
    const float* src = partial_row<D>(a.partial, all_rows, k, wid);
    const float4 e = *(const float4*)(src + D);
    if (e.y == -INFINITY && e.z == 0.f) continue;
    const float wo = ex2f(e.x - A), wl = ex2f(e.y - M);
    l += e.z * wl;
    if constexpr (D == 128) {
      const float4 x = *(const float4*)(src + lane * 4);
      acc[0] += x.x * wo; acc[1] += x.y * wo; acc[2] += x.z * wo; acc[3] += x.w * wo;
    } else {
      const float2 x = *(const float2*)(src + lane * 2);
      acc[0] += x.x * wo; acc[1] += x.y * wo;
    }
  }
  const float inv = l != 0.f ? exp2f(A - M) / l * (E4M3 ? 256.0f : 1.0f) : 0.f;
  const long long dst = (long long)row * a.o.st + (long long)head * a.o.sh + lane * (D / 32);
#pragma unroll
  for (int d = 0; d < D / 32; d += 2) {
    if constexpr (F32)
      *(float2*)((float*)a.o.p + dst + d) = make_float2(acc[d] * inv, acc[d + 1] * inv);
    else
      *(uint32_t*)((__nv_bfloat16*)a.o.p + dst + d) = pack_bf16x2(acc[d] * inv, acc[d + 1] * inv);
  }
}

template <int D, bool E4M3, bool F32>
cudaError_t launch(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  const int G = a.Hq / a.pool.Hkv;
  auto kern = kv_attn_kernel<D, E4M3, F32>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh<D>::BYTES);
  if (e != cudaSuccess) return e;
  const dim3 grid((unsigned)kv_places(a.batch.B, a.batch.T, G, 4, 1), (unsigned)a.pool.Hkv, (unsigned)plan.chunks);
  kern<<<grid, WARPS * 32, Sh<D>::BYTES, stream>>>(a, plan.chunk);
  e = cudaGetLastError();
  if (e != cudaSuccess) return e;
  ++*launches;
  if (plan.chunks > 1) {
    kv_join_kernel<D, E4M3, F32><<<(unsigned)(((long long)a.batch.T * a.Hq + 3) / 4), 128, 0, stream>>>(a, plan.chunk);
    e = cudaGetLastError();
    if (e == cudaSuccess) ++*launches;
  }
  return e;
}

}  // namespace

KvAttnPlan kv_attn_plan(const KvPool& pool, int B, int T, int dtype, int Hq, int max_length, int causal) {
  (void)dtype;
  (void)causal;
  const long long tiles = kv_places(B, T, Hq / pool.Hkv, 4, 1) * pool.Hkv;
  const long long want = (148 * 4 + tiles - 1) / tiles;
  const long long most = (max_length + 255) / 256;
  const long long chunks = want < most ? want : most;
  KvAttnPlan p;
  p.chunk = (int)(((max_length + chunks - 1) / chunks + 127) / 128 * 128);
  p.chunks = (int)((max_length + (long long)p.chunk - 1) / p.chunk);
  p.workspace = p.chunks > 1 ? sizeof(float) * (size_t)p.chunks * T * Hq * (pool.D + 4) : 0;
  return p;
}

cudaError_t launch_kv_attention(const KvAttnArgs& a, const KvAttnPlan& plan, cudaStream_t stream, int* launches) {
  const bool d128 = a.pool.D == 128, f32 = a.dtype == 0;
  if (a.pool.e4m3) {
    if (d128) return f32 ? launch<128, true, true>(a, plan, stream, launches) : launch<128, true, false>(a, plan, stream, launches);
    return f32 ? launch<64, true, true>(a, plan, stream, launches) : launch<64, true, false>(a, plan, stream, launches);
  }
  if (d128) return f32 ? launch<128, false, true>(a, plan, stream, launches) : launch<128, false, false>(a, plan, stream, launches);
  return f32 ? launch<64, false, true>(a, plan, stream, launches) : launch<64, false, false>(a, plan, stream, launches);
}

}  // namespace ar
