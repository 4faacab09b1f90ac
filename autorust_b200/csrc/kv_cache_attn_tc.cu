// Attention of many rows over the 8-bit paged cache (chunks of a prompt, whole prompts): the products on the tcgen05 tensor
// cores.  The same mathematics as kv_cache_attn.cu, bf16 tensors only:
//
//   x = (q . kcode) * (c_row * s_k * log2(e) / sqrt(D)) + log2(s_v / v_ref),   P = 2^(x - m + 8),   O = sum P vcode,   l = sum P * v_ref / s_v,   o = v_ref O / l
//
// v_ref is the scale of the CTA's first page, held inside [2^-5, 2^20]: scales that an append writes are 2^-60 to 2^121, so that v_ref / s_v
// and the sums of 2^31 keys stay normal f32 numbers.  Beside a page of huge values P may vanish where the row's sum needs it, and in front of a large
// logit m's rounding is more than P has room for (the multiply-add takes it off the exact product): a CTA that has a V scale above 2^15 v_ref among its pages, or a K
// scale that with its rows' largest |q| may make a logit of 2^20, keeps references as pairs (logit, log2 of the V scale), takes them off logit and scale
// each, and sums 2^(logit - m + 8), exponentials of their own.  It looks through its pages while the first tiles are on their way.  The scales of a page's keys and values are constants of a column block, so they ride on the multiply-add in front of the
// exponential, and the tensor cores see the codes as f16 (exact) and P and q in f16 (q scaled by a power of two per row:
// exact but for elements 2^-14 below its largest; P rounded to nearest, the row sum keeps the unrounded values).
//
// CTA = 2 tiles of 128 rows (tokens x query heads of the group) of one kv head, five warpgroups:
//   0, 1  softmax of tile 0 and 1: one thread per row = TMEM lane
//   2, 3  producers of K and of V: codes from global memory to f16 tiles in shared memory, rings of 2 tiles of 128 keys.  A
//         16-byte piece of codes becomes 32 bytes of a row; rows of 128 bytes in boxes of 64 channels, the 16-byte chunk c of
//         row r at c ^ (r & 7), as a swizzled TMA load would leave them: K is read K-major, V MN-major.  The next tile's codes
//         are in registers while the ring is full.
//   4     warps 0 and 1 issue the MMAs of tile 0 and 1: a wait that is over at once, a commit and the way to the next MMA take an
//         issuer some 400 clocks a step, under which the other's MMAs run (one issuer for both: 637 us of the case below)
//   TMEM (512 columns): S_0, S_1, O_0, O_1.  S_t is two buffers of 64 keys: while the softmax works on one, the other is computed,
// so that no row waits for the way from its weights over PV and QK to the next scores.  P (f16) overwrites the first half of its
// scores.  Step i of tile t: P_t(i) done -> O_t += P_t(i) V(i), then S_t(i + 2) = Q_t K(i + 2) into the same buffer.
// A row's O may be rescaled only when no PV of its tile is under way: the softmax waits for the last one then, which is rare.
//
// Measured, 2 x 1024 rows x 4 heads against 16384 keys, D = 128: 579 us, 920 TFLOP/s (573 before there were references as pairs; 1250 where they are taken).  S in one buffer of 128 keys took 643 us with one
// issuer and 674 with two.  With the softmax and the producers switched off (a scratch build) the MMAs and their hand-overs
// alone take 555: a step's 48 MMAs 85 clocks each, against 32 to 64 of arithmetic.  A buffer's round -- PV and QK of both tiles
// 1400 clocks, the way to the softmax 300, the softmax 1700, the way back 300 -- is what a step waits for; TMEM has room for two
// buffers per tile and no more.
#include <cuda_bf16.h>

#include "ar_ptx.cuh"
#include "kv_cache.cuh"
#include "softmax_math.cuh"

#include <type_traits>

namespace ar {
namespace {
using namespace arptx;

#ifdef AR_WAIT_TEST
__device__ int g_test_skip_cache_tile = -1;
__device__ int g_test_late_ns[3] = {0, 0, 0};
#endif

constexpr int BM = 128, BN = 128, HALF = 64, TILES = 2, ROWS = BM * TILES;
constexpr int THREADS = 640, W_PROD = 8, W_MMA = 16;
constexpr int SOFTMAX_REGS = 144, PRODUCER_REGS = 64, MMA_REGS = 64, LAUNCH_REGS = 96;
static_assert(256 * SOFTMAX_REGS + 256 * PRODUCER_REGS + 128 * MMA_REGS <= LAUNCH_REGS * THREADS, "register pool of the CTA");
constexpr int BLOCKS = BN / 16;  // column blocks of one page at least
constexpr float LOG2E = 1.4426950408889634f;
constexpr float P_SHIFT = 8.0f, LAG = 6.0f;  // P < 2^14: inside f16, and a weight 2^-22 of the largest still a normal number
constexpr float SCALE_FLOOR = 8.673617379884035e-19f;  // 2^-60
constexpr float V_REF_LEAST = 0.03125f, V_REF_MOST = 1048576.0f;
constexpr float WIDE = 32768.0f;  // s_v / v_ref
// Of 8 pairs of columns, those whose exponentials are the polynomial's (1.1e-4, below P's rounding to f16): the two tiles'
// softmax steps mostly fall together and share the MUFU (none 600 us of the case above, a quarter 576, three eighths 578, half 593).
constexpr uint32_t POLY_MASK = 0x88u;

template <int D>
struct Cfg {
  static constexpr int STAGES = 2;
  static constexpr int BOXES = D / 64;
  static constexpr int BOX = BN * 128;               // bytes: 128 rows of 64 channels
  static constexpr int TILE = BN * D * 2;            // of Q, K or V
  static constexpr int SCALE_RING = 4;               // tiles whose scales are kept
  static constexpr int NUM_BARS = 2 + 4 * STAGES + 4 + 4 + 4;
  static constexpr int SCALES = (TILES + 2 * STAGES) * TILE;
  static constexpr int BARS = SCALES + SCALE_RING * 3 * BLOCKS * 4;
  static constexpr int BYTES = BARS + NUM_BARS * 8 + 16 + 1024;
  static_assert(BYTES <= 227 * 1024, "shared memory budget");
  static constexpr uint32_t IDESC_QK = make_idesc(1, 0, 0, 0, 0, BM, HALF);  // f16 x f16 -> f32
  static constexpr uint32_t IDESC_PV = make_idesc(1, 0, 0, 0, 1, BM, D);
  static constexpr int QK_STEPS = D / 16, PV_STEPS = HALF / 16;
};

// x * 2^d, d <= 0, where 2^d by itself may be below the f32 numbers and x * 2^d is not.
__device__ __forceinline__ float times_ex2(float x, float d) { return x * ex2f(fmaxf(d, -100.0f)) * ex2f(fminf(d + 100.0f, 0.0f)); }
// Whether `some` holds in one of the 256 threads of the softmax, all of which come here.
__device__ __forceinline__ bool softmax_any(bool some) {
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"((uint32_t)some) : "memory");
  return __shfl_sync(0xffffffffu, any, 0) != 0;
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// Four codes -> two f16x2.  INT8: the byte code + 128 under the exponent of 1024 is 1152 + code.
template <bool E4M3>
__device__ __forceinline__ void expand4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
  } else {
    const uint32_t u = w ^ 0x80808080u, a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(0x64806480u));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(0x64806480u));
  }
}

// One arrival for the whole warp: 32 lanes that arrive one by one take the barrier's word in turn, 128 of them several hundred
// clocks (the handshakes of a step alone: 245 us of the case below).
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if (elect_one()) mbar_arrive(bar);
}

// SPLIT: the keys are divided over gridDim.z CTAs, which leave partial results for kv_join_rows_kernel: one row of D + 4 values per
// part, packed row and head -- the accumulated values, then m + log2 v_ref, m, l, or where the CTA was far, which the sign of l tells,
// m, m's part of the scale, -l, log2 v_ref.
template <int D, bool E4M3, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1) kv_attn_tc_kernel(const KvAttnArgs a, uint32_t* status, uint32_t ticket) {
  using C = Cfg<D>;
  constexpr int ST = C::STAGES;
  const float unit = (1.0f / sqrtf((float)D)) * LOG2E;  // of a logit in the log2 domain
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;
  uint8_t* sK = sQ + TILES * C::TILE;
  uint8_t* sV = sK + ST * C::TILE;
  float* scales = (float*)(smem + C::SCALES);  // [slot][s_k log2(e) / sqrt(D) | log2(s_v / v_ref) | v_ref / s_v][block]
  uint64_t* bars = (uint64_t*)(smem + C::BARS);
  uint64_t* q_full = bars;             // [2]
  uint64_t* k_full = q_full + 2;       // [ST]
  uint64_t* k_empty = k_full + ST;
  uint64_t* v_full = k_empty + ST;
  uint64_t* v_empty = v_full + ST;
  uint64_t* s_full = v_empty + ST;     // [tile][buffer]
  uint64_t* p_full = s_full + 4;       // [tile][buffer]
  uint64_t* pv_done = p_full + 4;      // [tile][buffer], each for one PV: the last of its buffer
  uint32_t* tmem_slot = (uint32_t*)(pv_done + 4);
  volatile uint32_t* abort_flag = tmem_slot + 1;
  uint32_t* tops = tmem_slot + 2;      // [2]: bits of the rows' largest |q|, of the pages' largest K scale
  const WaitCtx wctx{abort_flag, status, a.batch.sticky, ticket};

  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");  // whatever came before in the stream is done and visible

  const int tid = threadIdx.x;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const int lane = tid & 31;
  const int G = a.Hq / a.pool.Hkv, Hkv = a.pool.Hkv, h = blockIdx.y;
  // the last tiles first: under a causal mask they are the heavy ones
  KvPlace p = kv_place(a.batch, (int)(gridDim.x - 1 - blockIdx.x), G, 8, 1);
  // Read from memory, but the same for all threads: told to the compiler, which otherwise takes what follows for divergent and wraps
  // every tcgen05 instruction in an election of its own.
  p.b = __shfl_sync(0xffffffffu, p.b, 0);
  p.tile = __shfl_sync(0xffffffffu, p.tile, 0);
  p.row0 = __shfl_sync(0xffffffffu, p.row0, 0);
  p.n = __shfl_sync(0xffffffffu, p.n, 0);
  p.length = __shfl_sync(0xffffffffu, p.length, 0);
  const int all_rows = p.n * G;
  if (p.tile < 0 || (long long)p.tile * ROWS >= all_rows) return;
  const int r0 = p.tile * ROWS;
  const long long cap = min((long long)a.batch.table_pages << a.pool.page_log2, (long long)a.max_length);
  const int total = (int)min((long long)p.length, cap), pos0 = p.length - p.n;
  auto limit = [&](int row) { return a.causal ? max(min(total, pos0 + row / G + 1), 0) : total; };
  if (total < p.length && tid == 0) kv_report(a.batch);
  int end = limit(min(r0 + ROWS, all_rows) - 1), kb = 0;  // this CTA's keys: [kb, end)
  if constexpr (SPLIT) {
    const int tiles = (end + BN - 1) / BN;
    kb = (int)((long long)tiles * blockIdx.z / gridDim.z) * BN;
    end = min(end, (int)((long long)tiles * (blockIdx.z + 1) / gridDim.z) * BN);
  }
  int nh[2], low[2];  // halves of key tiles that some row of a row tile sees here; keys that all of them see
#pragma unroll
  for (int t = 0; t < TILES; t++) {
    const int first = r0 + t * BM, last = min(first + BM, all_rows) - 1;
    nh[t] = first > last ? 0 : (max(min(limit(last), end) - kb, 0) + HALF - 1) / HALF;
    low[t] = first > last ? 0 : limit(first);
  }
  const int nh_max = max(nh[0], nh[1]), nkv_max = (nh_max + 1) / 2;
  const int log2 = a.pool.page_log2;
  const int* table = a.batch.page_table + (long long)p.b * a.batch.table_stride;
  auto page_of = [&](int key) {  // -2: past the end, -1: there is none
    if (key >= end) return -2;
    const int pg = table[key >> log2];
    return pg >= 0 && pg < a.pool.pages ? pg : -1;
  };
  auto v_scale_of = [&](int pg) {
    const float s = a.pool.v_scale[(long long)pg * Hkv + h];
    return s < SCALE_FLOOR ? SCALE_FLOOR : s;  // (a NaN stays)
  };
  auto v_reference = [&]() {
    const int pg = page_of(kb);
    const float s = pg >= 0 ? v_scale_of(pg) : 1.0f;
    return s == s ? fminf(fmaxf(s, V_REF_LEAST), V_REF_MOST) : 1.0f;
  };

  bool lost = false;
  if (warp == W_MMA) {
    if (lane == 0) {
      lost = launch_lost(status, ticket);
      *abort_flag = lost ? 1u : 0u;
      tops[0] = tops[1] = 0u;
      for (int i = 0; i < 2; i++) {
        mbar_init(&q_full[i], 4);
        mbar_init(&s_full[2 * i], 1);
        mbar_init(&s_full[2 * i + 1], 1);
        mbar_init(&p_full[2 * i], 4);
        mbar_init(&p_full[2 * i + 1], 4);
        mbar_init(&pv_done[2 * i], 1);
        mbar_init(&pv_done[2 * i + 1], 1);
      }
      for (int i = 0; i < ST; i++) {
        mbar_init(&k_full[i], 4);
        mbar_init(&k_empty[i], TILES);
        mbar_init(&v_full[i], 4);
        mbar_init(&v_empty[i], TILES);
      }
      fence_mbar_init();
    }
    __syncwarp();
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tb = *tmem_slot;

  if (warp >= W_PROD && warp < W_MMA) {
    // ------------------------------------------------------------ producers: the first warpgroup K, the second V
    setmaxnreg_dec<PRODUCER_REGS>();
    const bool is_v = warp >= W_PROD + 4;
    const int ptid = tid & 127;
    constexpr int PIECES = D / 16;          // 16-byte pieces of a key's codes
    constexpr int PER = BN * PIECES / 128;  // of a tile, per thread
    constexpr int KEYS = 128 / PIECES;      // keys of one pass: 16 (D = 128) or 32; thread: key key_t of them, piece q
    const int key_t = ptid / PIECES, q = ptid % PIECES;
    const int in_page = (1 << log2) - 1;
    const long long page_bytes = ((long long)Hkv << log2) * D;
    const uint8_t* codes = (is_v ? a.pool.v : a.pool.k) + ((long long)h << log2) * D + (key_t & 15) * D + q * 16;
    const float v_ref = nkv_max > 0 ? v_reference() : 1.0f;
    // page numbers: lane l < 8 of every warp holds that of the tile's l-th block of 16 keys, two tiles ahead
    auto look = [&](int j) { return lane < BLOCKS ? page_of(kb + j * BN + lane * 16) : -2; };
    int pages = look(0), pages1 = look(1);
    uint4 held[PER];
    auto load = [&](int j, int pages) {
      const bool whole = __all_sync(0xffffffffu, pages >= 0 || lane >= BLOCKS) && kb + j * BN + BN <= end;
      if (whole && log2 == 7) {  // one page
        const uint8_t* src = codes + (long long)__shfl_sync(0xffffffffu, pages, 0) * page_bytes + (key_t & ~15) * D;
#pragma unroll
        for (int i = 0; i < PER; i++) held[i] = *(const uint4*)(src + i * KEYS * D);
      } else {
#pragma unroll
        for (int i = 0; i < PER; i++) {
          const int blk = (i * KEYS + key_t) >> 4;
          const int pg = __shfl_sync(0xffffffffu, pages, blk);
          const uint8_t* src = codes + (long long)pg * page_bytes + ((j * BN + blk * 16) & in_page) * D;
          held[i] = make_uint4(0u, 0u, 0u, 0u);  // keys past the end and without a page: codes of value 0
          if (pg >= 0 && kb + j * BN + i * KEYS + key_t < end) held[i] = *(const uint4*)src;
        }
      }
    };
    // Chunks 2 * (q & 3) and the next one of box q >> 2; the second box's pieces are written in the other order, so that the 8
    // lanes of a row write 8 different chunk places at a time.
    const int flip = (q >> 2) & 1;
    const uint32_t row_at = (q >> 2) * C::BOX + key_t * 128;
    const uint32_t at0 = row_at + ((((q & 3) * 2 + flip) ^ (key_t & 7)) << 4), at1 = row_at + ((((q & 3) * 2 + 1 - flip) ^ (key_t & 7)) << 4);
    auto store = [&](uint8_t* tile) {
#pragma unroll
      for (int i = 0; i < PER; i++) {
        const uint4 w = held[i];
        uint4 x, y;
        expand4<E4M3>(flip ? w.z : w.x, x.x, x.y);
        expand4<E4M3>(flip ? w.w : w.y, x.z, x.w);
        expand4<E4M3>(flip ? w.x : w.z, y.x, y.y);
        expand4<E4M3>(flip ? w.y : w.w, y.z, y.w);
        *(uint4*)(tile + at0 + i * KEYS * 128) = x;
        *(uint4*)(tile + at1 + i * KEYS * 128) = y;
      }
    };
    if (nkv_max > 0) load(0, pages);
    uint64_t *full = is_v ? v_full : k_full, *empty = is_v ? v_empty : k_empty;
    uint8_t* ring = is_v ? sV : sK;
    bool ok = !*abort_flag;
    for (int j = 0; j < nkv_max; j++) {
      const int s = j % ST, n = j / ST;
      const int now = pages;
      pages = pages1;
      pages1 = look(j + 2);
#ifdef AR_WAIT_TEST
      // Test build only: one tile is never delivered, so that the wait for it runs out.
      if (j == g_test_skip_cache_tile && !is_v) break;
      if (g_test_late_ns[is_v] > 0) __nanosleep(g_test_late_ns[is_v]);  // or every one comes late
#endif
      if (n > 0) ok = mbar_wait(&empty[s], (n - 1) & 1, wctx, is_v ? 0x51 : 0x50);
      if (!__all_sync(0xffffffffu, ok)) break;
      store(ring + s * C::TILE);
      if (!is_v && ptid < BLOCKS) {  // (lanes 0 .. 7 of the first warp, which hold the pages of their blocks)
        float* slot = scales + (j % C::SCALE_RING) * 3 * BLOCKS + ptid;
        float sk = 0.f, lv = -INFINITY, wv = 0.f;  // nothing there: every logit -inf, every weight 0
        if (now >= 0) {
          sk = a.pool.k_scale[(long long)now * Hkv + h] * unit;
          const float vs = v_scale_of(now);
          lv = log2f(vs) - log2f(v_ref);
          wv = vs == vs ? v_ref / vs : 1.0f;
        } else if (now == -1) {
          kv_report(a.batch);
        }
        slot[0] = sk;
        slot[BLOCKS] = lv;
        slot[2 * BLOCKS] = wv;
      }
      fence_proxy_async_smem();
      warp_arrive(&full[s]);
      if (j + 1 < nkv_max) load(j + 1, pages);
    }
  } else if (warp >= W_MMA) {
    setmaxnreg_dec<MMA_REGS>();
    if (warp < W_MMA + TILES) {
      // ---------------------------------------------------------- MMA issuers (converged; one elected lane issues)
      const int t = warp - W_MMA, mine = t ? nh[1] : nh[0];
      const uint64_t k_proto = make_sdesc_sw128(0, 16, 1024), v_proto = make_sdesc_sw128(0, C::BOX, 1024);
      const uint32_t k_hi = (uint32_t)(k_proto >> 32), v_hi = (uint32_t)(v_proto >> 32);
      const uint32_t q_lo = ((uint32_t)k_proto | (smem_u32(sQ) >> 4)) + t * (C::TILE >> 4);
      const uint32_t k_lo0 = (uint32_t)k_proto | (smem_u32(sK) >> 4);
      const uint32_t v_lo0 = (uint32_t)v_proto | (smem_u32(sV) >> 4);
      const uint32_t ts = tb + t * 128, to = tb + 256 + t * 128;
      // half i of the keys lies eight row groups of 1024 bytes into each box of tile i / 2
      auto issue_qk = [&](int i) {
        const uint32_t ka = k_lo0 + ((i >> 1) % ST) * (C::TILE >> 4) + (i & 1) * (HALF * 128 >> 4);
        if (!elect_one()) return;
#pragma unroll
        for (int x = 0; x < C::QK_STEPS; x++) {  // 16 channels = 32 bytes of a row, four to a box
          const uint32_t off = ((x >> 2) * C::BOX + (x & 3) * 32) >> 4;
          mma_ss_lohi<KIND_F16>(ts + (i & 1) * HALF, q_lo + off, k_hi, ka + off, k_hi, C::IDESC_QK, x > 0);
        }
      };
      auto issue_pv = [&](int i) {
        const uint32_t va = v_lo0 + ((i >> 1) % ST) * (C::TILE >> 4) + (i & 1) * (HALF * 128 >> 4);
        if (!elect_one()) return;
#pragma unroll
        for (int x = 0; x < C::PV_STEPS; x++)  // 16 keys = 2048 bytes of each box
          mma_ts_lohi<KIND_F16>(to, ts + (i & 1) * HALF + x * 8, va + x * (2048 >> 4), v_hi, C::IDESC_PV, (i > 0 || x > 0) ? 1u : 0u);
      };
      auto tile_in = [&](uint64_t* full, int j, uint32_t site) { return __all_sync(0xffffffffu, mbar_wait(&full[j % ST], (j / ST) & 1, wctx, site)); };
      bool ok = true;
      if (nh_max > 0) ok = tile_in(k_full, 0, 0x52);
      if (ok && mine > 0) ok = __all_sync(0xffffffffu, mbar_wait(&q_full[t], 0, wctx, 0x53));
      if (ok) {
        tc_fence_after();
        for (int i = 0; i < min(mine, 2); i++) {
          issue_qk(i);
          commit_one(&s_full[2 * t + i]);
        }
        if (nh_max > 0) commit_one(&k_empty[0]);
      }
      // (a row tile that sees fewer keys than the other passes on what it does not use)
      for (int i = 0; i < nh_max && ok; i++) {
        const int j = i >> 1, buf = i & 1;
        if (buf == 0) {  // a new tile of V, and of K for the step after next
          ok = tile_in(v_full, j, 0x54);
          if (j + 1 < nkv_max) ok = ok && tile_in(k_full, j + 1, 0x55);
          if (!ok) break;
        }
        if (i < mine) {
          ok = __all_sync(0xffffffffu, mbar_wait(&p_full[2 * t + buf], j & 1, wctx, 0x56));
          if (!ok) break;
          tc_fence_after();
          issue_pv(i);
          if (i + 2 < mine) {
            issue_qk(i + 2);
            commit_one(&s_full[2 * t + buf]);
          } else {
            commit_one(&pv_done[2 * t + buf]);
          }
        }
        if (buf == 1) {
          commit_one(&v_empty[j % ST]);
          if (j + 1 < nkv_max) commit_one(&k_empty[(j + 1) % ST]);
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax: thread = row
    setmaxnreg_inc<SOFTMAX_REGS>();
    const int t = warp >> 2, r = tid & 127, row = r0 + t * BM + r;
    const bool in = row < all_rows;
    const int token = in ? row / G : 0;
    const int lim = (in ? limit(row) : 0) - kb;
    const uint32_t lane_base = (uint32_t)(warp & 3) * 32;
    const uint32_t tS = tmem_addr(tb, lane_base, t * 128), tO = tmem_addr(tb, lane_base, 256 + t * 128);
    const int head = h * G + (in ? row - token * G : 0);

    // a huge V scale somewhere, the largest K scale
    bool far = false;
    float s_most = 0.f;
    uint32_t q_top = 0;
    if (nkv_max > 0) {
      const float most = WIDE * v_reference();
#pragma unroll 4
      for (int blk = (kb >> log2) + tid; blk <= (end - 1) >> log2; blk += 256) {
        const int pg = table[blk];
        if (pg >= 0 && pg < a.pool.pages) {
          far = far || a.pool.v_scale[(long long)pg * Hkv + h] > most;
          s_most = fmaxf(s_most, a.pool.k_scale[(long long)pg * Hkv + h]);  // (passes over NaN)
        }
      }
    }

    // Q: the row times 2^-e, its largest element below 2
    float c_row = 0.f;
    if (nh[t] > 0) {
      const uint4* src = (const uint4*)((const __nv_bfloat16*)a.q.p + (p.row0 + (long long)token) * a.q.st + (long long)head * a.q.sh);
      uint4 w[D / 8];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 8; i++) {
        w[i] = in ? src[i] : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
        for (int x = 0; x < 4; x++) top = max(top, max(u[x] << 16 & 0x7fffffffu, u[x] & 0x7fff0000u));
      }
      const bool odd = top >= 0x7f800000u;  // such a row is NaN: zeros here, a NaN sum at the end
      if (!odd) q_top = top;
      const int e = kv_binade(top);
      const float down = kv_power(-e);
      c_row = odd ? 0.f : kv_power(e);
      uint8_t* dst = sQ + t * C::TILE + r * 128;
#pragma unroll
      for (int i = 0; i < D / 8; i++) {
        if (odd) w[i] = make_uint4(0u, 0u, 0u, 0u);
        const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
        uint32_t v[4];
#pragma unroll
        for (int x = 0; x < 4; x++) v[x] = pack_half2(__uint_as_float(u[x] << 16) * down, __uint_as_float(u[x] & 0xffff0000u) * down);
        *(uint4*)(dst + (i >> 3) * C::BOX + (((i & 7) ^ (r & 7)) << 4)) = make_uint4(v[0], v[1], v[2], v[3]);
      }
      fence_proxy_async_smem();
      warp_arrive(&q_full[t]);
    }
    q_top = __reduce_max_sync(0xffffffffu, q_top);
    const uint32_t s_top = __reduce_max_sync(0xffffffffu, __float_as_uint(s_most));
    if (lane == 0) {
      atomicMax(&tops[0], q_top);
      atomicMax(&tops[1], s_top);
    }
    float m = -INFINITY, l = 0.f, me = 0.f;  // the reference is 2^(m + me), me 0 but in FARS
    float ref = 0.f;                         // what is taken off a logit: m - P_SHIFT, in FARS m; 0 as long as there is no m

    // One step: S of 64 keys -> P.  EDGE: keys from first_out on are not the row's; FAR: that, and scales or logits are far
    // apart.  False: a wait has run out.
    enum Kind { PLAIN, EDGES, FARS };
    auto step = [&](auto kind, int i) {
      constexpr bool EDGE = decltype(kind)::value != PLAIN, FAR = decltype(kind)::value == FARS;
      const float* slot = scales + ((i >> 1) % C::SCALE_RING) * 3 * BLOCKS + (i & 1) * (BLOCKS / 2);
      const int first_out = lim - i * HALF;
      const uint32_t ts = tS + (i & 1) * HALF;
      uint32_t sv[2][32];
      tmem_ld32(ts, sv[0]);
      tmem_ld32(ts + 32, sv[1]);
      const float4 sc = *(const float4*)slot, sa = *(const float4*)(slot + BLOCKS), sw = *(const float4*)(slot + 2 * BLOCKS);
      float c[4] = {c_row * sc.x, c_row * sc.y, c_row * sc.z, c_row * sc.w};
#pragma unroll
      for (int b = 0; b < 4; b++) c[b] = FAR && c[b] > KV_MOST_FACTOR * unit ? __uint_as_float(0x7fc00000u) : c[b];
      const float add[4] = {sa.x, sa.y, sa.z, sa.w};
      const float weight[4] = {sw.x, sw.y, sw.z, sw.w};
      tmem_wait_ld32(sv[0]);
      tmem_wait_ld32(sv[1]);
      float mc = -INFINITY;
      KvRef far_mc{-INFINITY, 0.f};
#pragma unroll
      for (int b = 0; b < 4; b++) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int x = 0; x < 16; x += 4) {
          float v[4];
#pragma unroll
          for (int k = 0; k < 4; k++) {
            v[k] = __uint_as_float(sv[b >> 1][(b & 1) * 16 + x + k]);
            if (EDGE && b * 16 + x + k >= first_out) v[k] = -INFINITY;
          }
          top[0] = fmax3(top[0], v[0], v[1]);
          top[1] = fmax3(top[1], v[2], v[3]);
        }
        // (a block without a page: s_k = 0 and log2 -inf; where all of it is hidden as well, 0 * -inf is NaN, which the
        // maximum passes over)
        if constexpr (FAR) {
          const float x = fmaxf(top[0], top[1]) * c[b];
          if (x > -INFINITY && add[b] > -INFINITY) far_mc = kv_larger(KvRef{x, add[b]}, far_mc);
        } else {
          mc = fmaxf(mc, fmaf(fmaxf(top[0], top[1]), c[b], add[b]));
        }
      }
      const bool need = FAR ? far_mc.m != -INFINITY && (m == -INFINITY || kv_over(far_mc, KvRef{m, me}) > LAG) : mc > m + LAG;
      if (__any_sync(0xffffffffu, need)) {
        float by = 0.f;  // log2 of what O and l are multiplied by
        if (need) by = m == -INFINITY ? -INFINITY : FAR ? kv_over(KvRef{m, me}, far_mc) : m - mc;
        const float alpha = ex2f(by);
        l = FAR ? times_ex2(l, by) : l * alpha;
        if (need) {
          m = FAR ? far_mc.m : mc;
          ref = FAR ? m : m - P_SHIFT;
          if (FAR) me = far_mc.e;
        }
        if (i > 0) {  // PV(i - 1) is done when S(i + 1), issued after it, is there; behind the last scores it reports itself
          const bool last = i + 1 == nh[t];
          uint64_t* bar = (last ? pv_done : s_full) + 2 * t + ((i + 1) & 1);
          if (!__all_sync(0xffffffffu, mbar_wait(bar, last ? 0 : ((i + 1) >> 1) & 1, wctx, 0x59))) return false;
          tc_fence_after();
          const uint64_t alpha2 = pack_f32x2(alpha, alpha);
#pragma unroll 1
          for (int cch = 0; cch < D / 16; cch++) {
            uint32_t ov[16];
            tmem_ld16(tO + cch * 16, ov);
            tmem_wait_ld();
#pragma unroll
            for (int x = 0; x < 16; x += 2) {
              float y, z;
              unpack_f32x2(mul_f32x2(pack_f32x2(__uint_as_float(ov[x]), __uint_as_float(ov[x + 1])), alpha2), y, z);
              ov[x] = __float_as_uint(y);
              ov[x + 1] = __float_as_uint(z);
            }
            tmem_st16(tO + cch * 16, ov);
          }
        }
      }
      if constexpr (FAR) {  // the scores become distances from the logit of the reference
#pragma unroll
        for (int b = 0; b < 4; b++) {
          float sum = 0.f;
#pragma unroll
          for (int x = 0; x < 16; x++) {
            uint32_t& s = sv[b >> 1][(b & 1) * 16 + x];
            const float d = __fmul_rn(__uint_as_float(s), c[b]) - ref;
            s = __float_as_uint(d);
            if (b * 16 + x < first_out) sum += ex2f(d + (P_SHIFT - me));
          }
          if (add[b] != -INFINITY) l += sum;
        }
      }
#pragma unroll
      for (int hf = 0; hf < 2; hf++) {
        uint32_t pk[16];
#pragma unroll
        for (int b2 = 0; b2 < 2; b2++) {
          const int b = hf * 2 + b2;
          const float by = FAR ? 1.0f : c[b], ab = FAR ? add[b] + (P_SHIFT - me) : add[b] - ref;
          const uint64_t c2 = pack_f32x2(by, by), add2 = pack_f32x2(ab, ab);
          uint64_t sum = pack_f32x2(0.f, 0.f);
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const int at = b2 * 16 + 2 * k;
            float p0, p1;
            const uint64_t x2 = fma_f32x2(pack_f32x2(__uint_as_float(sv[hf][at]), __uint_as_float(sv[hf][at + 1])), c2, add2);
            if (!EDGE && ((POLY_MASK >> k) & 1u))
              exp2_poly_x2(x2, p0, p1);
            else
              exp2_mufu_x2(x2, p0, p1);
            if constexpr (EDGE) {
              if (hf * 32 + at >= first_out) p0 = 0.f;
              if (hf * 32 + at + 1 >= first_out) p1 = 0.f;
            }
            sum = add_f32x2(sum, pack_f32x2(p0, p1));
            pk[b2 * 8 + k] = pack_half2(p0, p1);
          }
          float s0, s1;
          unpack_f32x2(sum, s0, s1);
          if (!FAR) l = fmaf(s0 + s1, weight[b], l);
        }
        tmem_st16(ts + hf * 16, pk);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&p_full[2 * t + (i & 1)]);
      return true;
    };

    auto scores = [&](int i) {  // false: a wait has run out
      const bool in = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * t + (i & 1)], (i >> 1) & 1, wctx, 0x57));
#ifdef AR_WAIT_TEST
      if (in && g_test_late_ns[2] > 0) __nanosleep(g_test_late_ns[2]);  // Test build only: every step comes late, as do the last products.
#endif
      tc_fence_after();
      return in;
    };
    bool ok = true;
    far = softmax_any(far);  // (tops are there, too)
    far = far || __uint_as_float(tops[1]) * __uint_as_float(tops[0] & 0x7f800000u) > KV_LARGE_LOGIT;
    if (!far) {
      for (int i = 0; i < nh[t] && ok; i++) {
        ok = scores(i);
        if (!ok) break;
        ok = kb + i * HALF + HALF > low[t] || kb + i * HALF + HALF > end ? step(std::integral_constant<Kind, EDGES>{}, i)
                                                                         : step(std::integral_constant<Kind, PLAIN>{}, i);
      }
    } else {
      for (int i = 0; i < nh[t] && ok; i++) ok = scores(i) && step(std::integral_constant<Kind, FARS>{}, i);
    }
    if (ok && nh[t] > 0) {
#ifdef AR_WAIT_TEST
      if (g_test_late_ns[2] > 0) __nanosleep(g_test_late_ns[2]);
#endif
      // the last two PV report on a barrier each: both may be under way or done, and a parity does not count phases
      ok = __all_sync(0xffffffffu, mbar_wait(&pv_done[2 * t + ((nh[t] - 1) & 1)], 0, wctx, 0x58));
      if (nh[t] > 1) ok = ok && __all_sync(0xffffffffu, mbar_wait(&pv_done[2 * t + (nh[t] & 1)], 0, wctx, 0x58));
      tc_fence_after();
    }
    if (ok) {
      if (c_row == 0.f && l > 0.f) l = __uint_as_float(0x7fc00000u);  // a q that is not finite, and a key that it sees
      const float v_ref = nh[t] > 0 ? v_reference() : 1.0f;
      const float inv = SPLIT ? 1.0f : nh[t] > 0 && l != 0.f ? v_ref / l : 0.f;
      __nv_bfloat16* dst = (__nv_bfloat16*)a.o.p + (p.row0 + (long long)token) * a.o.st + (long long)head * a.o.sh;
      float* part = a.partial + (((long long)blockIdx.z * a.batch.T + p.row0 + token) * a.Hq + head) * (D + 4);
#pragma unroll
      for (int cch = 0; cch < D / 32; cch++) {
        uint32_t ov[32];
        if (nh[t] > 0) {
          tmem_ld32(tO + cch * 32, ov);
          tmem_wait_ld();
        }
        if (in) {
#pragma unroll
          for (int i = 0; i < 8; i++) {
            float4 w = make_float4(0.f, 0.f, 0.f, 0.f);  // a row tile that sees no key
            if (nh[t] > 0)
              w = make_float4(__uint_as_float(ov[4 * i]) * inv, __uint_as_float(ov[4 * i + 1]) * inv, __uint_as_float(ov[4 * i + 2]) * inv,
                              __uint_as_float(ov[4 * i + 3]) * inv);
            if constexpr (SPLIT)
              *(float4*)(part + cch * 32 + i * 4) = w;
            else
              *(uint2*)(dst + cch * 32 + i * 4) = make_uint2(pack_bf16x2(w.x, w.y), pack_bf16x2(w.z, w.w));
          }
        }
      }
      if (SPLIT && in) *(float4*)(part + D) = far ? make_float4(m, me, -l, log2f(v_ref)) : make_float4(m + log2f(v_ref), m, l, 0.f);
    }
  }
  // ---------------------------------------------------------------- teardown
  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) tmem_dealloc(tb, 512);
}

// o = 2^(A - M) sum_p 2^(A_p - A) O_p / sum_p 2^(m_p - M) l_p over the parts of a row, in order; A_p = m_p + log2 v_ref_p.  One warp per
// packed row and head.
constexpr int MOST_PARTS = 16;
constexpr float NEG = -1e30f;  // below every m of a part that is not far (2^20), but -inf, which there is none of
template <int D>
__device__ __forceinline__ void store_row(__nv_bfloat16* dst, const float (&x)[D / 32], float inv) {
#pragma unroll
  for (int d = 0; d < D / 32; d += 2) *(uint32_t*)(dst + d) = pack_bf16x2(x[d] * inv, x[d + 1] * inv);
}
// A row of which some part is far: references as distances from the largest logit among them.  `src`: the lane's values of part 0, `entry`
// the row's entry in it, `next` from part to part.
template <int D>
__device__ __noinline__ void join_far_row(const float* src, const float* entry, long long next, int parts, __nv_bfloat16* dst) {
  constexpr int V = D / 32;
  auto row = [&](int p) {  // {m, m's part of the scale, l, log2 v_ref}
    const float4 e = *(const float4*)(entry + p * next);
    if (__float_as_uint(e.z) >> 31) return make_float4(e.x, e.y, -e.z, e.w);
    return make_float4(e.y, 0.f, e.z, e.y == -INFINITY ? 0.f : e.x - e.y);
  };
  float top = -INFINITY, A = -INFINITY, M = -INFINITY, l = 0.f;
  for (int p = 0; p < parts; p++) top = fmaxf(top, row(p).x);
  const float base = top == -INFINITY ? 0.f : top;
  for (int p = 0; p < parts; p++) {
    const float4 e = row(p);
    M = fmaxf(M, (e.x - base) + e.y);
    A = fmaxf(A, (e.x - base) + (e.y + e.w));
  }
  float x[V];
#pragma unroll
  for (int d = 0; d < V; d++) x[d] = 0.f;
  for (int p = 0; p < parts; p++) {
    const float4 e = row(p);
    const bool none = e.x == -INFINITY;  // zeros, or in a row of NaN a NaN sum: 0 * NaN is wanted
    const float wo = none ? 0.f : ex2f((e.x - base) + (e.y + e.w) - A);
    l += times_ex2(e.z, none ? -INFINITY : (e.x - base) + e.y - M);
#pragma unroll
    for (int d = 0; d < V; d++) x[d] = fmaf(src[p * next + d], wo, x[d]);
  }
  store_row<D>(dst, x, l != 0.f ? exp2f(A - M) / l : 0.f);
}
template <int D>
__global__ void __launch_bounds__(256) kv_join_rows_kernel(const KvAttnArgs a, int parts) {
  asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const long long rows = (long long)a.batch.T * a.Hq, at = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (at >= rows) return;
  const int row = (int)(at / a.Hq), head = (int)(at - (long long)row * a.Hq);
  const KvPlace p = kv_place(a.batch, row, 1, 0, 0);
  if (row < p.row0 || row >= p.row0 + p.n) return;  // a row of no sequence
  constexpr int V = D / 32;
  float4 e[MOST_PARTS];
  float A = NEG, M = NEG;
  uint32_t signs = 0;
#pragma unroll
  for (int i = 0; i < MOST_PARTS; i++) {
    e[i] = make_float4(NEG, NEG, 0.f, 0.f);
    if (i < parts) e[i] = *(const float4*)(a.partial + (i * rows + at) * (D + 4) + D);
    A = fmaxf(A, e[i].x);
    M = fmaxf(M, e[i].y);
    signs |= __float_as_uint(e[i].z);
  }
  __nv_bfloat16* dst = (__nv_bfloat16*)a.o.p + (long long)row * a.o.st + (long long)head * a.o.sh + lane * V;
  if (signs >> 31) {
    const float* entry = a.partial + at * (D + 4) + D;
    join_far_row<D>(entry - D + lane * V, entry, rows * (D + 4), parts, dst);
    return;
  }
  float x[V], l = 0.f;
#pragma unroll
  for (int d = 0; d < V; d++) x[d] = 0.f;
#pragma unroll
  for (int i = 0; i < MOST_PARTS; i++) {
    if (i < parts) {
      const float* src = a.partial + (i * rows + at) * (D + 4) + lane * V;
      const float wo = ex2f(e[i].x - A);
      l += times_ex2(e[i].z, e[i].y - M);
#pragma unroll
      for (int d = 0; d < V; d += 2) {
        const float2 y = *(const float2*)(src + d);
        x[d] = fmaf(y.x, wo, x[d]);
        x[d + 1] = fmaf(y.y, wo, x[d + 1]);
      }
    }
  }
  store_row<D>(dst, x, l != 0.f ? exp2f(A - M) / l : 0.f);
}

template <int D, bool E4M3>
cudaError_t launch(const KvAttnArgs& a, int parts, cudaStream_t stream, int* launches) {
  auto kern = parts > 1 ? kv_attn_tc_kernel<D, E4M3, true> : kv_attn_tc_kernel<D, E4M3, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::BYTES);
  if (e != cudaSuccess) return e;
  uint32_t *status = nullptr, ticket = 0;
  if (!launch_ticket(stream, &status, &ticket)) return cudaErrorUnknown;
  const dim3 grid((unsigned)kv_places(a.batch, a.Hq / a.pool.Hkv, 8, 1), (unsigned)a.pool.Hkv, (unsigned)parts);
  e = launch_early(kern, grid, dim3(THREADS), Cfg<D>::BYTES, stream, a, status, ticket);
  if (e != cudaSuccess) return e;
  ++*launches;
  if (parts > 1) {
    e = launch_early(kv_join_rows_kernel<D>, dim3((unsigned)(((long long)a.batch.T * a.Hq + 7) / 8)), dim3(256), 0, stream, a, parts);
    if (e == cudaSuccess) ++*launches;
  }
  return e;
}

}  // namespace

cudaError_t launch_kv_attention_tc(const KvAttnArgs& a, int parts, cudaStream_t stream, int* launches) {
  if (a.pool.e4m3) return a.pool.D == 128 ? launch<128, true>(a, parts, stream, launches) : launch<64, true>(a, parts, stream, launches);
  return a.pool.D == 128 ? launch<128, false>(a, parts, stream, launches) : launch<64, false>(a, parts, stream, launches);
}

}  // namespace ar

#ifdef AR_WAIT_TEST
// Test build only: which tile of keys the producers leave out, -1 for none; by how many nanoseconds those of K and V, and the rows at their end,
// come late.
extern "C" int ar_test_skip_cache_tile(int j) {
  return (int)cudaMemcpyToSymbol(ar::g_test_skip_cache_tile, &j, sizeof(int));
}
extern "C" int ar_test_late_cache_tiles(int k_ns, int v_ns, int rows_ns) {
  const int ns[3] = {k_ns, v_ns, rows_ns};
  return (int)cudaMemcpyToSymbol(ar::g_test_late_ns, ns, sizeof(ns));
}
#endif
