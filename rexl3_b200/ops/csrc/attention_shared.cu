// Paged GQA attention of a decode / verify window whose sequences share pages (sm_100a): the pages that neighbouring sequences have in common (a cached
// system prompt, a document that many streams ask about) are read once for all of them, the rest once per sequence.
//
//     out[r][h] = sum_j softmax_j(scale * q[r][h] . k_j) v_j over the keys j < ctx_len[r]; a row without keys gives 0
//
// The rows of the window are put into blocks: the (row, query head) pairs of one KV head, up to 128 of them, that see the same pages - rows of a group of
// sequences over the group's common pages, or rows of one sequence over its own.  128 pairs are the M of a tcgen05 MMA: S = Q K^T and O += P V run as in
// attention_tc.cu (page by page, S and P and O in tensor memory, thread = pair = TMEM lane), without a causal edge.  64 streams behind a prompt of 8192 tokens
// read its 33.5 MB per layer once instead of 64 times.
//
// All pages of all (block, KV head) units stand in one line, cut into equal pieces, one for each of 296 CTAs (two per SM): a CTA's piece may end in
// one unit and begin in another.  Each (unit, CTA) leaves partial outputs in fp32 with their maxima and sums, and a merge kernel joins a row's in a fixed order.
// Where the pieces end depends on the whole window, and with it the order of a row's sum: unlike attn_decode's, a row's last bits depend on its window mates.
//
// Warps: 0 = TMA producer, 1 = MMA issuer (owns the tensor memory), 2..5 = softmax, for E4M3 caches 6..7 = expansion of byte pages to fp16 operand tiles.
// All waits are bounded (status words), no cluster multicast.
#include <cuda.h>
#include <cuda_fp8.h>
#include <type_traits>
#include "common.cuh"

namespace rx {

constexpr int SH_PAGE = 64, SH_PAIRS = 128, SH_CTAS = 296, SH_MAX_ROWS = 1024;
constexpr int SH_MIN_SHARED = 1;                        // pages that a group must have in common

// ------------------------------------------------------------------------------------------------ plan
// Layout (int32): [0] pages of all units  [1] pages per CTA  [2] blocks  [3] n_kv, then the block at which each CTA begins, the blocks, and per row its
// block over common pages, its block over own pages (-1: none), the keys it sees and nothing.
struct ShBlock {
  int row, rows;          // first row, rows
  int seq;                // table row
  int page, pages;        // first page, pages
  int before;             // pages of the blocks before (times n_kv: where the block's units begin in the line)
  int part;               // partial vectors (times n_q) of the blocks before
  int most;               // keys that some row of the block's group sees: what stands behind them is never multiplied
};
static_assert(sizeof(ShBlock) == 32, "two 16-byte loads");
constexpr int SH_HEAD = 8, SH_AT_BLOCKS = SH_HEAD + ((SH_CTAS + 7) / 8) * 8;
constexpr int SH_AT_ROWS = SH_AT_BLOCKS + 2 * SH_MAX_ROWS * 8;
constexpr int SH_PLAN_INTS = SH_AT_ROWS + 4 * SH_MAX_ROWS + 4;      // (with room to align it)

__device__ __forceinline__ int sh_slots(int pages, int L) { return (pages + L - 1) / L + 1; }      // CTAs that a unit of `pages` pages can meet

// inclusive sum over the block's threads; `all` gets the total
__device__ __forceinline__ int block_scan(int v, int* s_warp, int& all) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int p = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += p;
  }
  if (lane == 31) s_warp[warp] = v;
  __syncthreads();
  int w = lane < nw ? s_warp[lane] : 0;
  const int mine = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int p = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += p;
  }
  all = __shfl_sync(0xffffffffu, w, 31);
  v += __shfl_sync(0xffffffffu, w - mine, warp);
  __syncthreads();
  return v;
}

// Thread = row.  A run is the adjacent rows of one sequence.  Runs are joined into a group where their link (the pages that a run has in common with the one
// before it) is at least SH_MIN_SHARED pages and at least half of each neighbouring link: a group shares its smallest link, and one pair of
// strangers with nothing but a first page in common must not take a long prompt away from the pairs on both sides.
__global__ void __launch_bounds__(SH_MAX_ROWS) shared_plan_kernel(const int* __restrict__ row_seq, const int* __restrict__ ctx_len, const int* __restrict__ common,
                                                                  int rows, int n_tables, int width, int rt, int n_kv, int* __restrict__ plan, int* status) {
  pdl_launch();
  __shared__ int s_seq[SH_MAX_ROWS], s_first[SH_MAX_ROWS + 1], s_link[SH_MAX_ROWS + 1], s_group[SH_MAX_ROWS], s_shared[SH_MAX_ROWS], s_gfirst[SH_MAX_ROWS + 1],
      s_gmost[SH_MAX_ROWS], s_most[SH_MAX_ROWS], s_before[2 * SH_MAX_ROWS], s_warp[32];
  pdl_wait();
  const int r = threadIdx.x;
  const bool live = r < rows;
  int seq = live ? row_seq[r] : -1, ctx = live ? ctx_len[r] : 0;
  const int link = live ? min(max(common[r], 0), width) : 0;
  if (live && (seq < 0 || seq >= n_tables || ctx < 0 || ctx > (long long)width * SH_PAGE)) {
    set_status(status, ST_BAD_ARG, 95, r);
    ctx = 0;                                               // a row that sees nothing; without a table row it is a run of its own that nobody is linked to
    if (seq < 0 || seq >= n_tables) seq = -1 - r;
  }
  if (live) s_seq[r] = seq, s_shared[r] = 0x7FFFFFFF, s_gmost[r] = s_most[r] = 0;
  __syncthreads();
  int runs, groups, all;
  const bool head = live && (r == 0 || s_seq[r - 1] != seq);
  const int run = block_scan(head, s_warp, runs) - 1;
  if (head) s_first[run] = r, s_link[run] = r == 0 || seq < 0 || s_seq[r - 1] < 0 ? 0 : link;
  if (r == 0) s_first[runs] = rows, s_link[runs] = 0;
  __syncthreads();
  const int mine = r < runs ? s_link[r] : 0;               // (thread = run)
  const bool joined = r > 0 && r < runs && mine >= SH_MIN_SHARED && 2 * (long long)mine >= s_link[r - 1] && 2 * (long long)mine >= s_link[r + 1];
  const int g_of_run = block_scan(r < runs && !joined, s_warp, groups) - 1;
  if (r < runs) {
    s_group[r] = g_of_run;
    if (!joined) s_gfirst[g_of_run] = s_first[r];
  }
  if (r == 0) s_gfirst[groups] = rows;
  __syncthreads();
  if (joined) atomicMin(&s_shared[g_of_run], mine);
  const int group = live ? s_group[run] : 0, first = live ? s_first[run] : 0;
  const int chunk = first + (r - first) / rt * rt;         // first row of the row's block over its own pages
  if (live) {
    atomicMax(&s_gmost[group], ctx);
    atomicMax(&s_most[chunk], ctx);
  }
  __syncthreads();
  const int shared = live && s_shared[group] != 0x7FFFFFFF ? min(s_shared[group], (s_gmost[group] + SH_PAGE - 1) / SH_PAGE) : 0;
  const int gfirst = live ? s_gfirst[group] : 0, tile = gfirst + (r - gfirst) / rt * rt;
  const int own = live ? max((s_most[chunk] + SH_PAGE - 1) / SH_PAGE - shared, 0) : 0;
  const bool lead_s = live && shared > 0 && r == tile, lead_o = live && own > 0 && r == chunk;
  int pages_s, pages_o, blocks;
  const int b_in = block_scan((lead_s ? 1 : 0) | (lead_o ? 1 << 16 : 0), s_warp, blocks);
  const int p_s = block_scan(lead_s ? shared : 0, s_warp, pages_s), p_o = block_scan(lead_o ? own : 0, s_warp, pages_o);
  const int nb_s = blocks & 0xFFFF, nb = nb_s + (blocks >> 16);
  const int total = (pages_s + pages_o) * n_kv, L = max((total + SH_CTAS - 1) / SH_CTAS, 1);
  const int n_s = live ? min(rt, s_gfirst[group + 1] - tile) : 0, n_o = live ? min(rt, s_first[run + 1] - chunk) : 0;
  const int v_s = block_scan(lead_s ? n_s * sh_slots(shared, L) : 0, s_warp, all);
  const int all_s = all;
  const int v_o = block_scan(lead_o ? n_o * sh_slots(own, L) : 0, s_warp, all);
  ShBlock* blk = reinterpret_cast<ShBlock*>(plan + SH_AT_BLOCKS);
  // (s_seq and s_link are free: the ids of the blocks that begin at a row)
  __syncthreads();
  if (lead_s) {
    const int id = (b_in & 0xFFFF) - 1;
    s_link[r] = id, s_before[id] = p_s - shared;
    blk[id] = ShBlock{r, n_s, s_seq[gfirst], 0, shared, p_s - shared, v_s - n_s * sh_slots(shared, L), s_gmost[group]};
  }
  __syncthreads();
  if (lead_o) {
    const int id = nb_s + (b_in >> 16) - 1;
    s_seq[r] = id, s_before[id] = pages_s + p_o - own;
    blk[id] = ShBlock{r, n_o, seq, shared, own, pages_s + p_o - own, all_s + v_o - n_o * sh_slots(own, L), s_most[chunk]};
  }
  __syncthreads();
  if (live) {
    reinterpret_cast<int4*>(plan + SH_AT_ROWS)[r] = make_int4(shared > 0 ? s_link[tile] : -1, own > 0 ? s_seq[chunk] : -1, ctx, 0);
  }
  for (int c = r; c < SH_CTAS; c += blockDim.x) {
    int lo = 0, hi = nb - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)s_before[mid] * n_kv <= (long long)c * L) lo = mid; else hi = mid - 1;
    }
    plan[SH_HEAD + c] = lo;
  }
  if (r == 0) plan[0] = total, plan[1] = L, plan[2] = nb, plan[3] = n_kv;
}

// ------------------------------------------------------------------------------------------------ attention
__device__ __forceinline__ void sh_ld_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
      "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ float sh_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two probabilities as one operand word: bf16 beside a bf16 cache, fp16 beside an expanded one (both operands of an MMA have one type)
template <bool F16>
__device__ __forceinline__ uint32_t sh_pack(float lo, float hi) {
  if constexpr (F16) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
// V page as the B operand: keys x head_dim with the head dimension contiguous (MN-major, 128-byte swizzle; see attention_tc.cu)
__device__ __forceinline__ uint64_t sh_desc_v(uint32_t smem_addr) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

struct ShArgs {
  const uint16_t* q;
  const int* block_table;
  const int* plan;
  const float* kv_scale;
  float* part_o;
  float* part_ml;
  int* status;
  int max_blocks, n_q, n_kv;
  float scale_log2;
};

template <int HD, bool F8>
struct Sh {
  static constexpr int TILE = SH_PAGE * HD * 2, RAW = SH_PAGE * HD, QBOX = SH_PAIRS * 128;
  static constexpr int KS = F8 ? 1 : 2, VS = F8 ? 1 : 2, RS = 2;            // stages of K, of V, of byte pages
  static constexpr int OPERANDS = (KS + VS) * TILE, RAWS = F8 ? 2 * RS * RAW : 0, Q = HD / 64 * QBOX;
  static constexpr int SMEM = OPERANDS + RAWS + Q + 256 + 1024;
  static constexpr int THREADS = F8 ? 256 : 192;
  static constexpr int S_COLS = 64, O = 128;                                // tensor memory: two S buffers of 64 columns | O
  static constexpr int COLS = 256;
};

// a wait's outcome for the whole warp: what follows it is done by all lanes or by none
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok); }

struct ShSegment { ShBlock b; int kvh, page, pages, slot, slots; };          // a CTA's pages of one unit
// The CTA's piece of the line as segments; every role walks it by itself.
struct ShWalk {
  const ShBlock* blk;
  int b, pos, end, L, n_kv;
  __device__ __forceinline__ ShWalk(const int* plan, int n_kv_) : n_kv(n_kv_) {
    const int total = plan[0];
    L = plan[1];
    blk = reinterpret_cast<const ShBlock*>(plan + SH_AT_BLOCKS);
    pos = (int)min((long long)total, (long long)blockIdx.x * L), end = (int)min((long long)total, (long long)pos + L);
    b = plan[SH_HEAD + blockIdx.x];
  }
  __device__ __forceinline__ bool next(ShSegment& s) {
    if (pos >= end) return false;
    const int4* p = reinterpret_cast<const int4*>(blk + b);
    int4 x = p[0], y = p[1];
    int rel = pos - y.y * n_kv;
    if (rel >= y.x * n_kv) {                                                // the block is done
      p = reinterpret_cast<const int4*>(blk + ++b);
      x = p[0], y = p[1];
      rel = pos - y.y * n_kv;
    }
    s.b = ShBlock{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
    s.kvh = rel / s.b.pages, s.page = rel - s.kvh * s.b.pages;
    s.pages = min(end - pos, s.b.pages - s.page);
    const int unit = s.b.before * n_kv + s.kvh * s.b.pages;
    s.slot = (int)blockIdx.x - unit / L, s.slots = sh_slots(s.b.pages, L);
    pos += s.pages;
    return true;
  }
};

template <int HD, bool F8>
__global__ void __launch_bounds__((Sh<HD, F8>::THREADS), 2)
attn_shared_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ ShArgs a) {
  using C = Sh<HD, F8>;
  constexpr int TILE = C::TILE, BOXES = HD / 64;
  pdl_launch();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* k_sm = smem;                                   // [stage][box (64 d)][64 keys][128 B]
  uint8_t* v_sm = smem + C::KS * TILE;
  uint8_t* q_sm = smem + C::OPERANDS;                     // [box][128 pairs][128 B]
  uint8_t* raw = q_sm + C::Q;                             // [stage][K, V][64 keys][HD]
  uint64_t* bars = (uint64_t*)(raw + C::RAWS);
  uint64_t* k_full = bars;                                // [KS] the copy, or both expanding warps
  uint64_t* v_full = k_full + 2;
  uint64_t* k_empty = v_full + 2;                         // commit after QK
  uint64_t* v_empty = k_empty + 2;                        // commit after PV
  uint64_t* s_full = v_empty + 2;                         // [2] commit after QK
  uint64_t* p_ready = s_full + 2;                         // [2] the 4 softmax warps
  uint64_t* pv_done = p_ready + 2;                        // [1] commit after PV
  uint64_t* q_ready = pv_done + 1;                        // [1] the 4 softmax warps, once per segment
  uint64_t* drained = q_ready + 1;
  uint64_t* raw_full = drained + 1;                       // [RS]
  uint64_t* raw_empty = raw_full + 2;                     // [RS] both expanding warps
  uint32_t* tmem_slot = (uint32_t*)(raw_empty + 2);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], F8 ? 2 : 1); mbar_init(&v_full[i], F8 ? 2 : 1); mbar_init(&k_empty[i], 1); mbar_init(&v_empty[i], 1);
      mbar_init(&s_full[i], 1); mbar_init(&p_ready[i], 4); mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 2);
    }
    mbar_init(pv_done, 1); mbar_init(q_ready, 4); mbar_init(drained, 1);
    *abort_flag = 0;
    fence_barrier_init();
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();                                             // the plan, q and the caches were written by the previous kernels
  const uint32_t tmem_base = *tmem_slot;
  const int G = a.n_q / a.n_kv;
  ShWalk walk(a.plan, a.n_kv);
  ShSegment sg;

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA producer
    if (elect_one()) {
      int n = 0, n_v = 0;                                 // pages (bf16: of K, of V) issued
      bool ok = true;
      while (ok && walk.next(sg)) {
        const int* bt = a.block_table + (size_t)sg.b.seq * a.max_blocks + sg.b.page + sg.page;
        for (int j = 0; j < sg.pages && ok; ++j) {
          const int y = (bt[j] * a.n_kv + sg.kvh) * SH_PAGE;
          if constexpr (F8) {
            const int st = n % C::RS;
            if (n >= C::RS) ok = mbar_wait(&raw_empty[st], ((n / C::RS) - 1) & 1, abort_flag, a.status, 96, 100);
            if (!ok) break;
            mbar_arrive_expect_tx(&raw_full[st], 2 * C::RAW);
            tma_load_2d(raw + st * 2 * C::RAW, &tk, 0, y, &raw_full[st]);
            tma_load_2d(raw + st * 2 * C::RAW + C::RAW, &tv, 0, y, &raw_full[st]);
            ++n;
          } else {
            const int st = n % C::KS;
            if (n >= C::KS) ok = mbar_wait(&k_empty[st], ((n / C::KS) - 1) & 1, abort_flag, a.status, 96, 100);
            if (!ok) break;
            mbar_arrive_expect_tx(&k_full[st], TILE);
            for (int x = 0; x < BOXES; ++x) tma_load_2d(k_sm + st * TILE + x * 8192, &tk, x * 64, y, &k_full[st]);
            ++n;
            if (n_v >= C::VS) ok = mbar_wait(&v_empty[st], ((n_v / C::VS) - 1) & 1, abort_flag, a.status, 97, 100);
            if (!ok) break;
            mbar_arrive_expect_tx(&v_full[st], TILE);
            for (int x = 0; x < BOXES; ++x) tma_load_2d(v_sm + st * TILE + x * 8192, &tv, x * 64, y, &v_full[st]);
            ++n_v;
          }
        }
      }
      if constexpr (F8) ring_landed(raw_full, C::RS, n);
      else {
        ring_landed(k_full, C::KS, n);
        ring_landed(v_full, C::VS, n_v);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t fmt = F8 ? 0 : 1;
      constexpr uint32_t idesc_qk = umma_idesc_f16(SH_PAIRS, SH_PAGE, fmt, fmt);              // both K-major
      constexpr uint32_t idesc_pv = umma_idesc_f16(SH_PAIRS, HD, fmt, fmt) | (1u << 16);      // B (V) is MN-major
      const uint64_t qd = umma_desc_k_sw128(smem_u32(q_sm));
      int done = 0, segs = 0;                             // pages and segments before this one
      bool ok = true;
      // S = Q K(j)^T of the CTA's page `n` into buffer n & 1
      auto qk = [&](int n) {
        const int st = n % C::KS;
        if (!mbar_wait(&k_full[st], (n / C::KS) & 1, abort_flag, a.status, 98)) return false;
        tc_fence_after();
        const uint64_t kd = umma_desc_k_sw128(smem_u32(k_sm + st * TILE));
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
          tc_mma_f16(tmem_base + (n & 1) * C::S_COLS, qd + (uint64_t)((kk >> 2) * (C::QBOX >> 4) + (kk & 3) * 2), kd + (uint64_t)((kk >> 2) * (8192 >> 4) + (kk & 3) * 2),
                     idesc_qk, kk != 0);
        tc_commit(&s_full[n & 1]);
        tc_commit(&k_empty[st]);
        return true;
      };
      while (ok && walk.next(sg)) {
        ok = mbar_wait(q_ready, segs & 1, abort_flag, a.status, 99);
        for (int j = 0; j < 2 && j < sg.pages && ok; ++j) ok = qk(done + j);
        for (int j = 0; j < sg.pages && ok; ++j) {
          const int n = done + j, st = n % C::VS;
          ok = mbar_wait(&v_full[st], (n / C::VS) & 1, abort_flag, a.status, 100) && mbar_wait(&p_ready[n & 1], (n >> 1) & 1, abort_flag, a.status, 101);
          if (!ok) break;
          tc_fence_after();
          const uint32_t vbase = smem_u32(v_sm + st * TILE);
#pragma unroll
          for (int kk = 0; kk < SH_PAGE / 16; ++kk)
            tc_mma_f16_ts(tmem_base + C::O, tmem_base + (n & 1) * C::S_COLS + kk * 8, sh_desc_v(vbase + kk * 2048), idesc_pv, (j | kk) != 0);
          tc_commit(pv_done);
          tc_commit(&v_empty[st]);
          if (j + 2 < sg.pages) ok = qk(n + 2);           // overwrites P(n) after PV(n) has read it (a thread's MMAs run in issue order)
        }
        done += sg.pages;
        ++segs;
      }
      // every MMA issued so far has completed when this commit arrives: the columns may then be returned
      tc_commit(drained);
      for (int i = 0; i < (1 << 22) && !mbar_try_wait(drained, 0); ++i) {}   // bounded, and not cut short by the abort word
    }
  } else if (warp < 6) {
    // ---------------------------------------------------------------- softmax warps: thread = (row, head) pair = TMEM lane
    const int quarter = warp & 3, pair = quarter * 32 + lane;
    const uint32_t lane_addr = tmem_base + ((uint32_t)(quarter * 32) << 16);
    int done = 0;
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int rb = pair / G, hq = sg.kvh * G + pair % G;
      const bool live = rb < sg.b.rows, some = quarter * 32 < sg.b.rows * G;   // (uniform) the warp holds a pair
      const int row = sg.b.row + (live ? rb : 0);
      const int keys = live ? a.plan[SH_AT_ROWS + 4 * row + 2] : 0;     // keys the pair sees
      if (some) {
        // q -> shared memory: 128-byte rows, 16-byte chunk c of a box at c ^ (row & 7).  The MMAs that read the segment before's have completed: this
        // warp has seen the scores of its last page.
        const uint4* src = reinterpret_cast<const uint4*>(a.q + ((size_t)row * a.n_q + (live ? hq : 0)) * HD);
        uint8_t* dst = q_sm + pair * 128;
#pragma unroll
        for (int i = 0; i < HD / 8; ++i) {
          uint4 v = live ? __ldg(src + i) : make_uint4(0u, 0u, 0u, 0u);
          if constexpr (F8) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int u = 0; u < 4; ++u) w[u] = sh_pack<true>(__uint_as_float(w[u] << 16), __uint_as_float(w[u] & 0xFFFF0000u));
          }
          *reinterpret_cast<uint4*>(dst + (i >> 3) * C::QBOX + (((i & 7) ^ (pair & 7)) << 4)) = v;
        }
        fence_proxy_async();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_ready);
      const float scale_log2 = F8 ? a.scale_log2 * a.kv_scale[sg.kvh] : a.scale_log2;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < sg.pages && ok; ++j) {
        const int n = done + j;
        const uint32_t s_addr = lane_addr + (n & 1) * C::S_COLS;
        ok = all_ok(mbar_wait(&s_full[n & 1], (n >> 1) & 1, abort_flag, a.status, 102));
        if (!ok) break;
        const int key0 = (sg.b.page + sg.page + j) * SH_PAGE;
        if (some) {
          tc_fence_after();
          uint32_t s0[32], s1[32];
          sh_ld_x32(s_addr, s0);
          sh_ld_x32(s_addr + 32, s1);
          tc_wait_ld();
          if (key0 + SH_PAGE > keys) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              if (key0 + i >= keys) s0[i] = 0xFF800000u;
              if (key0 + 32 + i >= keys) s1[i] = 0xFF800000u;
            }
          }
          float mx = -INFINITY;
#pragma unroll
          for (int i = 0; i < 32; ++i) mx = fmaxf(mx, fmaxf(__uint_as_float(s0[i]), __uint_as_float(s1[i])));
          const float ms = mx * scale_log2;
          float alpha = 1.f;
          // the running maximum moves only by more than 2^8: the probabilities stay below 2^8, harmless in 16-bit operands and fp32 sums
          if (ms > m + 8.f || m == -INFINITY) {
            const float m_new = fmaxf(m, ms);
            alpha = (m == -INFINITY) ? 1.f : sh_ex2(m - m_new);
            m = m_new;
          }
          const float m_use = (m == -INFINITY) ? 0.f : m;
          float lsum = 0.f;
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float pa = sh_ex2(fmaf(__uint_as_float(s0[2 * i]), scale_log2, -m_use));
            const float pb = sh_ex2(fmaf(__uint_as_float(s0[2 * i + 1]), scale_log2, -m_use));
            const float pc = sh_ex2(fmaf(__uint_as_float(s1[2 * i]), scale_log2, -m_use));
            const float pd = sh_ex2(fmaf(__uint_as_float(s1[2 * i + 1]), scale_log2, -m_use));
            lsum += (pa + pb) + (pc + pd);
            pk[i] = sh_pack<F8>(pa, pb);
            pk[16 + i] = sh_pack<F8>(pc, pd);
          }
          tc_st_32x32b_x32(s_addr, pk);
          l = l * alpha + lsum;
          if (j > 0) {                                    // O was last written by the PV before: rescale it where a pair's maximum moved
            ok = all_ok(mbar_wait(pv_done, (n - 1) & 1, abort_flag, a.status, 103));
            if (!ok) break;
            tc_fence_after();
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll
              for (int ch = 0; ch < HD / 32; ++ch) {
                uint32_t r[32];
                sh_ld_x32(lane_addr + C::O + ch * 32, r);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                tc_st_32x32b_x32(lane_addr + C::O + ch * 32, r);
              }
            }
          }
          tc_wait_st();
          tc_fence_before();
        }
        // Keys that no row sees yet: their V may hold anything, and 0 * NaN would reach every pair
        if (key0 + SH_PAGE > sg.b.most) {
          ok = all_ok(mbar_wait(&v_full[n % C::VS], (n / C::VS) & 1, abort_flag, a.status, 104));
          if (!ok) break;
          uint8_t* v = v_sm + (n % C::VS) * TILE;
          for (int i = max(sg.b.most - key0, 0) * 8 + (warp - 2) * 32 + lane; i < SH_PAGE * 8; i += 128)
#pragma unroll
            for (int x = 0; x < BOXES; ++x) *reinterpret_cast<uint4*>(v + x * 8192 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async();
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[n & 1]);
      }
      done += sg.pages;
      if (!ok) break;
      ok = all_ok(mbar_wait(pv_done, (done - 1) & 1, abort_flag, a.status, 105));
      if (!ok) break;
      if (some) {
        tc_fence_after();
        const float v_scale = F8 ? a.kv_scale[a.n_kv + sg.kvh] : 1.f;
        const size_t at = (size_t)(sg.b.part + rb * sg.slots + sg.slot) * a.n_q + hq;
        float4* dst = reinterpret_cast<float4*>(a.part_o + at * HD);
#pragma unroll
        for (int ch = 0; ch < HD / 32; ++ch) {
          uint32_t r[32];
          sh_ld_x32(lane_addr + C::O + ch * 32, r);
          tc_wait_ld();
          if (live) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[ch * 8 + i] = make_float4(__uint_as_float(r[4 * i]) * v_scale, __uint_as_float(r[4 * i + 1]) * v_scale, __uint_as_float(r[4 * i + 2]) * v_scale,
                                            __uint_as_float(r[4 * i + 3]) * v_scale);
          }
        }
        if (live) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(m, l);
        tc_fence_before();                                // the reads of O are ordered before the next segment's first PV by q_ready / p_ready
      }
    }
  } else if constexpr (F8) {
    // ---------------------------------------------------------------- expansion of byte pages: E4M3 -> fp16 (exact) in the operand layout
    const int tid = threadIdx.x - 192;
    constexpr int CHUNKS = C::RAW / 16;
    auto expand = [&](const uint8_t* src, uint8_t* dst) {
#pragma unroll 4
      for (int c = tid; c < CHUNKS; c += 64) {
        const int key = c / (HD / 16), x = c % (HD / 16);
        const uint4 b = lds128(smem_u32(src) + c * 16);
        const uint32_t w[4] = {b.x, b.y, b.z, b.w};
        uint32_t h[8];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(h[2 * i]), "=r"(h[2 * i + 1]) : "r"(w[i]));
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int ch = 2 * x + u;                       // 16-byte chunk of the fp16 row
          *reinterpret_cast<uint4*>(dst + (ch >> 3) * 8192 + key * 128 + (((ch & 7) ^ (key & 7)) << 4)) = make_uint4(h[4 * u], h[4 * u + 1], h[4 * u + 2], h[4 * u + 3]);
        }
      }
      fence_proxy_async();
      __syncwarp();
    };
    int n = 0;
    bool ok = true;
    while (ok && walk.next(sg)) {
      for (int j = 0; j < sg.pages && ok; ++j, ++n) {
        const int st = n % C::RS;
        ok = all_ok(mbar_wait(&raw_full[st], (n / C::RS) & 1, abort_flag, a.status, 106));
        if (ok && n >= C::KS) ok = all_ok(mbar_wait(&k_empty[n % C::KS], ((n / C::KS) - 1) & 1, abort_flag, a.status, 107));
        if (!ok) break;
        expand(raw + st * 2 * C::RAW, k_sm + (n % C::KS) * TILE);
        if (lane == 0) mbar_arrive(&k_full[n % C::KS]);
        if (n >= C::VS) ok = all_ok(mbar_wait(&v_empty[n % C::VS], ((n / C::VS) - 1) & 1, abort_flag, a.status, 108));
        if (!ok) break;
        expand(raw + st * 2 * C::RAW + C::RAW, v_sm + (n % C::VS) * TILE);
        if (lane == 0) {
          mbar_arrive(&v_full[n % C::VS]);
          mbar_arrive(&raw_empty[st]);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem_base, C::COLS);
}

// ------------------------------------------------------------------------------------------------ merge
// Joins a row's partial outputs, common pages before own, CTA by CTA: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  A warp per 128 outputs; with
// `suh` also xr = fp16(H(out * suh)), the input rotation of the output projection.
template <int HD>
__global__ void __launch_bounds__(128) attn_shared_merge_kernel(const int* plan, const float* part_o, const float* part_ml, int n_q, int n_kv,
                                                                const __half* __restrict__ suh, __half* __restrict__ xr, uint16_t* __restrict__ out) {
  pdl_launch();
  pdl_wait();
  const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, width = n_q * HD;
  const int b = blockIdx.y * 4 + warp;
  if (b >= width / 128) return;
  const int e0 = b * 128 + lane * 4, hq = e0 / HD, d0 = e0 % HD, kvh = hq / (n_q / n_kv), L = plan[1];
  const ShBlock* blk = reinterpret_cast<const ShBlock*>(plan + SH_AT_BLOCKS);
  size_t at[2] = {0, 0};
  int n[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int id = plan[SH_AT_ROWS + 4 * row + u];
    if (id < 0) continue;
    const ShBlock s = blk[id];
    const int unit = s.before * n_kv + kvh * s.pages;
    n[u] = (unit + s.pages - 1) / L - unit / L + 1;
    at[u] = (size_t)(s.part + (row - s.row) * sh_slots(s.pages, L)) * n_q + hq;
  }
  auto slot = [&](int s) { return s < n[0] ? at[0] + (size_t)s * n_q : at[1] + (size_t)(s - n[0]) * n_q; };
  const int all = n[0] + n[1];
  float m = -INFINITY;
  for (int s = 0; s < all; ++s) m = fmaxf(m, part_ml[slot(s) * 2]);
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f;
#pragma unroll 8
  for (int s = 0; s < all; ++s) {
    const size_t i = slot(s);
    const float2 ml = *reinterpret_cast<const float2*>(part_ml + i * 2);
    const float4 o = *reinterpret_cast<const float4*>(part_o + i * HD + d0);
    const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - m);
    l += f * ml.y;
    acc[0] += f * o.x, acc[1] += f * o.y, acc[2] += f * o.z, acc[3] += f * o.w;
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = all > 0 ? acc[i] * inv : 0.f;
  if (out != nullptr) *reinterpret_cast<uint2*>(out + (size_t)row * width + e0) = make_uint2(sh_pack<false>(acc[0], acc[1]), sh_pack<false>(acc[2], acc[3]));
  if (xr != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= __half2float(suh[e0 + i]);
    fwht128_warp(acc);
    *reinterpret_cast<uint2*>(xr + (size_t)row * width + e0) = make_uint2(sh_pack<true>(acc[0], acc[1]), sh_pack<true>(acc[2], acc[3]));
  }
}

template <int HD, bool F8>
static cudaError_t launch_shared(int dev, const CUtensorMap& tk, const CUtensorMap& tv, const ShArgs& a, cudaStream_t st) {
  static bool configured[64];
  if (dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_kernel<HD, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh<HD, F8>::SMEM);
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  return rx::launch(attn_shared_kernel<HD, F8>, dim3(SH_CTAS), dim3(Sh<HD, F8>::THREADS), Sh<HD, F8>::SMEM, st, tk, tv, a);
}

}  // namespace rx

using namespace rx;

RX_API int rx_attn_shared_plan_ints() { return SH_PLAN_INTS; }

// Partial vectors: a block of n rows meets at most pages / L + 2 CTAs per KV head, and all blocks' pages / L together at most SH_CTAS / n_kv; a row is in two blocks.
RX_API long long rx_attn_shared_scratch_floats(int rows, int n_q, int n_kv, int hd) {
  if (rows < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || n_q / n_kv > SH_PAIRS) return 0;
  const long long rt = SH_PAIRS / (n_q / n_kv), vectors = (rt * SH_CTAS / n_kv + 1 + 4ll * rows) * n_q;
  return vectors * (hd + 2) + SH_PLAN_INTS;
}

static bool sh_takes(int rows, int n_q, int n_kv, int n_tables, int max_blocks) {
  return rows >= 1 && rows <= SH_MAX_ROWS && n_kv >= 1 && n_q >= n_kv && n_q % n_kv == 0 && n_q / n_kv <= SH_PAIRS && n_tables >= 1 && max_blocks >= 1 &&
         (long long)rows * max_blocks * n_kv < (1ll << 29) && max_blocks < (1 << 24);
}

RX_API int rx_attn_shared_plan(const void* row_seq, const void* ctx_len, const void* common, int rows, int n_tables, int max_blocks, int n_q, int n_kv, void* plan,
                               int* status, void* stream) {
  if (!sh_takes(rows, n_q, n_kv, n_tables, max_blocks)) return (int)cudaErrorInvalidValue;
  const int threads = rows <= 128 ? 128 : (rows + 31) / 32 * 32;
  return (int)rx::launch(shared_plan_kernel, dim3(1), dim3(threads), 0, (cudaStream_t)stream, (const int*)row_seq, (const int*)ctx_len, (const int*)common, rows,
                         n_tables, max_blocks, SH_PAIRS / (n_q / n_kv), n_kv, (int*)plan, status);
}

// scratch: rx_attn_shared_scratch_floats floats, 16-byte aligned.  plan == nullptr: the call plans into the scratch.  kv_scale == nullptr: bf16 caches.
RX_API int rx_attn_shared(const void* tmap_k, const void* tmap_v, const void* q, const void* block_table, int n_tables, int max_blocks, const void* row_seq,
                          const void* ctx_len, const void* common, void* scratch, int rows, int n_q, int n_kv, int hd, float scale, const void* kv_scale,
                          const void* suh, void* xr, void* out, const void* plan, int* status, void* stream) {
  if (!sh_takes(rows, n_q, n_kv, n_tables, max_blocks) || (hd != 64 && hd != 128) || n_q * hd % 128 != 0 || (out == nullptr && xr == nullptr) ||
      (suh == nullptr) != (xr == nullptr))
    return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  const long long vectors = (rx_attn_shared_scratch_floats(rows, n_q, n_kv, hd) - SH_PLAN_INTS) / (hd + 2);
  ShArgs a;
  a.part_o = (float*)scratch; a.part_ml = a.part_o + vectors * hd;
  int* own_plan = (int*)(a.part_ml + vectors * 2);
  own_plan = (int*)(((uintptr_t)own_plan + 15) & ~(uintptr_t)15);
  a.q = (const uint16_t*)q; a.block_table = (const int*)block_table; a.plan = plan != nullptr ? (const int*)plan : own_plan;
  a.kv_scale = (const float*)kv_scale; a.status = status; a.max_blocks = max_blocks; a.n_q = n_q; a.n_kv = n_kv; a.scale_log2 = scale * 1.4426950408889634f;
  if (plan == nullptr) {
    const int r = rx_attn_shared_plan(row_seq, ctx_len, common, rows, n_tables, max_blocks, n_q, n_kv, own_plan, status, stream);
    if (r != 0) return r;
  }
  const CUtensorMap &tk = *(const CUtensorMap*)tmap_k, &tv = *(const CUtensorMap*)tmap_v;
  if (hd == 128) e = kv_scale != nullptr ? launch_shared<128, true>(dev, tk, tv, a, st) : launch_shared<128, false>(dev, tk, tv, a, st);
  else e = kv_scale != nullptr ? launch_shared<64, true>(dev, tk, tv, a, st) : launch_shared<64, false>(dev, tk, tv, a, st);
  if (e != cudaSuccess) return (int)e;
  return (int)rx::launch(hd == 128 ? attn_shared_merge_kernel<128> : attn_shared_merge_kernel<64>, dim3(rows, (n_q * hd / 128 + 3) / 4), dim3(128), 0, st, a.plan, a.part_o,
                         a.part_ml, n_q, n_kv, (const __half*)suh, (__half*)xr, (uint16_t*)out);
}
