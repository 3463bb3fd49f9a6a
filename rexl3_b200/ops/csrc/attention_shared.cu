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
// one unit and begin in another.  Each (unit, CTA) segment leaves partial outputs in fp32 with their maxima and sums, and a merge kernel joins a row's in a
// fixed order.  Where the pieces end depends on the whole window, and with it the order of a row's sum: unlike attn_decode's, a row's last bits depend on
// its window mates.
//
// A page's 64 scores a pair go to tensor memory, come back as exponentials in 16 bits over the same columns, and are the A operand of the product with V.
// The QKs run two pages ahead of the PVs, also into the next segment.  Scores, maxima, sums and outputs are fp32; the probabilities are rounded to the type that V
// has as an operand (both operands of an MMA have one), and their sum is that of the unrounded ones: each stands for itself within 2^-8 (bf16) or 2^-11 (fp16; in
// the range where that is exact to 11 bits, else within 2^-32 of the row's largest: see UP), no more than the rounding of the outputs.
//
// Warps: 0..3 = softmax, 4 = feeder (descriptions of the segments; TMA), 5 = MMA issuer (owns the tensor memory), for E4M3 caches 6, 7 and 8, 9 = expansion of
// byte pages of K and of V to fp16 operand tiles.
// A block of up to 64 or 32 pairs would leave two or three quarters idle and the others bound by one warp's exponentials: its queries
// stand among the 128 two or four times, each copy takes its part of a page's keys - the rest of its P is zero - and leaves its own partial output.
// All waits are bounded (status words), no cluster multicast.
//
// Whole calls with 40 query and 8 KV heads of 128, one after the other over the same cache, the plan (inside the kernel for up to 64 rows: 1.5 to 3 us) and the merge
// (4 to 5 us) included:
//     64 rows behind 8192 common keys, 60 .. 700 keys of their own: 44 us.  134 MB, 20.6 us at the rate of a copy.  Three blocks read each common page, so L2 gives 200 MB:
//         a page comes 3100 cycles after it is asked for and five are on their way to each CTA, 37 bytes a clock and SM or 9.7 TB/s of them all; the rest is the first
//         pages' way, the last CTAs' and the merge.
//     48 rows of 500 .. 4000 keys behind 150 common ones: 84 us.  448 MB, 68.6 us: bound by memory, 5.3 TB/s.
//     32 rows behind 32,700 common keys, E4M3: 65 us.  104 MB, 16 us: bound by instructions, the expansion's beside the softmax's (bf16: 208 MB, 60 us).
#include <cuda.h>
#include <cuda_fp8.h>
#include <type_traits>
#include "common.cuh"

namespace rx {

constexpr int SH_PAGE = 64, SH_PAIRS = 128, SH_CTAS = 296, SH_MAX_ROWS = 1024, SH_FUSED_ROWS = 64;
// Pages that a group must have in common.  (64 rows of 40 heads and 100 .. 700 keys: of one common page nothing comes either way, 3 pages 37.1 against 38.5 us where
// each sequence reads them for itself, 6 pages 37.4 against 40.6; 256 rows of 8 heads and up to 60 keys behind 3 pages 23.5 against 27 us.)
constexpr int SH_MIN_SHARED = 1;
// What a unit costs beside its pages, in pages: its place in the line is that much longer.  (One, two, three, four: 64 rows behind 8192 common keys 46.6, 44.2, 45.3,
// 47.5 us; 16 sequences of five rows behind 4001 28.7, 26.1, 25.6, 25.6; 32 E4M3 rows behind 32,700 69.4, 65.3, 65.7, 65.9; 48 rows of 500 .. 4000 keys 86.6, 84.4, 84.2, 85.1,
// of E4M3 112, 92, 81, 75: two is best for long common prompts, and E4M3 rows that share nothing would take more.  Pages weighted by the copies of their block's pairs,
// 8 : 7 : 6, changed as much for the worse as for the better.)
constexpr int SH_SEGMENT = 2;
// A CTA's piece has no least length: one of two or four pages leaves fewer partial outputs, but on 57 drawn windows of all sizes it gained nothing, or lost 7 %.
// Few warps of the merge would join many partial outputs one after the other, so up to 148 blocks of 128 outputs go by 16 warps each where a row may have more than 64
// (by the width of the table, the only bound that the host knows: a small window in a wide table takes 11.5 us by 16 warps, 10.4 in a narrow one by four),
// up to 1480 by four, more by one: two rows of five heads behind 31,637 keys, 992 partial outputs each, 90 -> 26 us of the whole call; 32 rows of 40 heads behind 32,700
// (1280 blocks of some 30) 70 -> 65 us; but 1728 blocks of few 24 -> 27 us by four, and four blocks of few 11.0 -> 12.7 us by 16.
constexpr int SH_SPLIT16 = 148, SH_SPLIT16_OF = 64, SH_SPLIT4 = 1480;

// ------------------------------------------------------------------------------------------------ plan
// Layout (int32): [0] length of the line  [1] a CTA's piece  [2] blocks  [3] n_kv  [4] n_q  [5] rows  [6] table rows  [7] pages of one, then the block at which each CTA begins, the blocks, per row what the merge
// asks of its block over common pages and of its block over own pages - length of the blocks before, pages (0: no block), the row's partial vectors, copies -,
// and the keys that each row sees.
struct ShBlock {
  int row, rows;          // first row; rows, and << 8 how many CTAs a unit can meet
  int seq;                // table row
  int page, pages;        // first page, pages
  int before;             // length of the blocks before (times n_kv: where the block's units begin in the line)
  int part;               // partial vectors (times n_q) of the blocks before
  int most;               // keys that some row of the block's group sees: what stands behind them is never multiplied
};
static_assert(sizeof(ShBlock) == 32, "two 16-byte loads");
constexpr int SH_HEAD = 8, SH_AT_BLOCKS = SH_HEAD + ((SH_CTAS + 7) / 8) * 8;
constexpr int SH_AT_ROWS = SH_AT_BLOCKS + 2 * SH_MAX_ROWS * 8;
constexpr int SH_AT_KEYS = SH_AT_ROWS + 8 * SH_MAX_ROWS, SH_PLAN_INTS = SH_AT_KEYS + SH_MAX_ROWS + 4;      // (with room to align it)

__device__ __forceinline__ int sh_slots(int pages, int L) { return (pages + L - 1) / L + 1; }      // CTAs that a unit of `pages` pages can meet
__device__ __forceinline__ int sh_copies(int pairs) { return pairs <= 32 ? 4 : pairs <= 64 ? 2 : 1; }
// where the pages of a unit begin in the line
__device__ __forceinline__ int sh_unit(int before, int pages, int kvh, int n_kv) { return before * n_kv + kvh * (pages + SH_SEGMENT) + SH_SEGMENT; }

// the plan is one of this shape of window: its blocks, pages and partial vectors are in bounds
__device__ __forceinline__ bool sh_fits(const int* plan, int n_kv, int n_q, int rows, int n_tables, int max_blocks) {
  const int4* head = reinterpret_cast<const int4*>(plan);
  const int4 x = head[0], y = head[1];
  return x.w == n_kv && y.x == n_q && y.y == rows && y.z == n_tables && y.w == max_blocks;
}

// inclusive sums over the block's threads, of N values each; `all` gets the totals
template <int N>
__device__ __forceinline__ void block_scan(int (&v)[N], int (*s_warp)[32], int (&all)[N]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int p = __shfl_up_sync(0xffffffffu, v[i], o);
      if (lane >= o) v[i] += p;
    }
  if (lane == 31)
#pragma unroll
    for (int i = 0; i < N; ++i) s_warp[i][warp] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    int w = lane < nw ? s_warp[i][lane] : 0;
    const int mine = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int p = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += p;
    }
    all[i] = __shfl_sync(0xffffffffu, w, 31);
    v[i] += __shfl_sync(0xffffffffu, w - mine, warp);
  }
  __syncthreads();
}

// Thread = row.  A run is the adjacent rows of one sequence.  Runs are joined into a group where their link (the pages that a run has in common with the one
// before it) is at least SH_MIN_SHARED pages and at least half of each neighbouring link: a group shares its smallest link, and one pair of
// strangers with nothing but a first page in common must not take a long prompt away from the pairs on both sides.
// Of up to MAX rows, by all threads of the block, at least as many; its thread `r` looks up the first blocks of the CTAs cta, cta + cta_step ...;
// `all`: what the merge asks, and the status, too.
template <int MAX>
struct ShPlan {
  int seq[MAX], first[MAX + 1], link[MAX + 1], group[MAX], shared[MAX], gfirst[MAX + 1], gmost[MAX], most[MAX], before[2 * MAX], warp[3][32];
};
template <int MAX>
__device__ __forceinline__ void sh_plan(ShPlan<MAX>& sh, const int* row_seq, const int* ctx_len, const int* common, int rows, int n_tables, int width, int G, int n_kv,
                                        int* plan, int* status, bool all, int cta, int cta_step) {
  int *s_seq = sh.seq, *s_first = sh.first, *s_link = sh.link, *s_group = sh.group, *s_shared = sh.shared, *s_gfirst = sh.gfirst, *s_gmost = sh.gmost, *s_most = sh.most,
      *s_before = sh.before, (*s_warp)[32] = sh.warp;
  const int r = threadIdx.x, rt = SH_PAIRS / G;
  const bool live = r < rows;
  int seq = live ? row_seq[r] : -1, ctx = live ? ctx_len[r] : 0;
  const int link = live ? min(max(common[r], 0), width) : 0;
  if (live && (seq < 0 || seq >= n_tables || ctx < 0 || ctx > (long long)width * SH_PAGE)) {
    if (all) set_status(status, ST_BAD_ARG, 95, r);
    ctx = 0;                                               // a row that sees nothing; without a table row it is a run of its own that nobody is linked to
    if (seq < 0 || seq >= n_tables) seq = -1 - r;
  }
  if (live) s_seq[r] = seq, s_shared[r] = 0x7FFFFFFF, s_gmost[r] = s_most[r] = 0;
  __syncthreads();
  const bool head = live && (r == 0 || s_seq[r - 1] != seq);
  int heads[1] = {head}, all_runs[1];
  block_scan(heads, s_warp, all_runs);
  const int run = heads[0] - 1, runs = all_runs[0];
  if (head) s_first[run] = r, s_link[run] = r == 0 || seq < 0 || s_seq[r - 1] < 0 ? 0 : link;
  if (r == 0) s_first[runs] = rows, s_link[runs] = 0;
  __syncthreads();
  const int mine = r < runs ? s_link[r] : 0;               // (thread = run)
  const bool joined = r > 0 && r < runs && mine >= SH_MIN_SHARED && 2 * (long long)mine >= s_link[r - 1] && 2 * (long long)mine >= s_link[r + 1];
  int leaders[1] = {r < runs && !joined}, all_groups[1];
  block_scan(leaders, s_warp, all_groups);
  const int g_of_run = leaders[0] - 1, groups = all_groups[0];
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
  const int len_s = shared + SH_SEGMENT, len_o = own + SH_SEGMENT;
  int sum[3] = {(lead_s ? 1 : 0) | (lead_o ? 1 << 16 : 0), lead_s ? len_s : 0, lead_o ? len_o : 0}, sums[3];
  block_scan(sum, s_warp, sums);
  const int b_in = sum[0], p_s = sum[1], p_o = sum[2], blocks = sums[0], pages_s = sums[1], pages_o = sums[2];
  const int nb_s = blocks & 0xFFFF, nb = nb_s + (blocks >> 16);
  const int total = (pages_s + pages_o) * n_kv, L = max((total + SH_CTAS - 1) / SH_CTAS, 1);
  const int n_s = live ? min(rt, s_gfirst[group + 1] - tile) : 0, n_o = live ? min(rt, s_first[run + 1] - chunk) : 0;
  const int k_s = n_s * sh_slots(shared, L) * sh_copies(n_s * G), k_o = n_o * sh_slots(own, L) * sh_copies(n_o * G);
  int vec[2] = {lead_s ? k_s : 0, lead_o ? k_o : 0}, vecs[2];
  block_scan(vec, s_warp, vecs);
  const int v_s = vec[0], v_o = vec[1], all_s = vecs[0];
  ShBlock* blk = reinterpret_cast<ShBlock*>(plan + SH_AT_BLOCKS);
  // (s_link and s_first, then s_seq and s_gfirst are free: length and partial vectors before the block that begins at a row)
  __syncthreads();
  if (lead_s) {
    const int id = (b_in & 0xFFFF) - 1;
    s_link[r] = s_before[id] = p_s - len_s, s_first[r] = v_s - k_s;
    blk[id] = ShBlock{r, n_s | sh_slots(shared, L) << 8, s_seq[gfirst], 0, shared, p_s - len_s, v_s - k_s, s_gmost[group]};
  }
  __syncthreads();
  if (lead_o) {
    const int id = nb_s + (b_in >> 16) - 1;
    s_seq[r] = s_before[id] = pages_s + p_o - len_o, s_gfirst[r] = all_s + v_o - k_o;
    blk[id] = ShBlock{r, n_o | sh_slots(own, L) << 8, seq, shared, own, pages_s + p_o - len_o, all_s + v_o - k_o, s_most[chunk]};
  }
  __syncthreads();
  if (live) {
    const int c_s = sh_copies(n_s * G), c_o = sh_copies(n_o * G);
    if (all) {
      int4* of = reinterpret_cast<int4*>(plan + SH_AT_ROWS) + 2 * r;
      of[0] = shared > 0 ? make_int4(s_link[tile], shared, s_first[tile] + (r - tile) * sh_slots(shared, L) * c_s, c_s) : make_int4(0, 0, 0, 0);
      of[1] = own > 0 ? make_int4(s_seq[chunk], own, s_gfirst[chunk] + (r - chunk) * sh_slots(own, L) * c_o, c_o) : make_int4(0, 0, 0, 0);
    }
    plan[SH_AT_KEYS + r] = ctx;
  }
  for (int c = cta; c < SH_CTAS; c += cta_step) {
    int lo = 0, hi = nb - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((long long)s_before[mid] * n_kv <= (long long)c * L) lo = mid; else hi = mid - 1;
    }
    plan[SH_HEAD + c] = lo;
  }
  if (r == 0) plan[0] = total, plan[1] = L, plan[2] = nb, plan[3] = n_kv, plan[4] = n_kv * G, plan[5] = rows, plan[6] = n_tables, plan[7] = width;
}
__global__ void __launch_bounds__(SH_MAX_ROWS) shared_plan_kernel(const int* row_seq, const int* ctx_len, const int* common, int rows, int n_tables, int width,
                                                                  int G, int n_kv, int* plan, int* status) {
  pdl_launch();
  __shared__ ShPlan<SH_MAX_ROWS> sh;
  pdl_wait();
  sh_plan(sh, row_seq, ctx_len, common, rows, n_tables, width, G, n_kv, plan, status, true, threadIdx.x, blockDim.x);
}
// The plan of a window of few rows, by each CTA of the attention for itself: all write the same words to the same places, and read what they have written.  (What only
// the merge reads is written by one.)
__device__ __noinline__ void sh_plan_here(void* smem, const int* row_seq, const int* ctx_len, const int* common, int rows, int n_tables, int width, int G, int n_kv, int* plan,
                                          int* status) {
  sh_plan(*reinterpret_cast<ShPlan<SH_FUSED_ROWS>*>(smem), row_seq, ctx_len, common, rows, n_tables, width, G, n_kv, plan, status, blockIdx.x == 0,
          threadIdx.x == 0 ? (int)blockIdx.x : SH_CTAS, SH_CTAS);
  fence_proxy_async();                                     // (the copies' places were the plan's)
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------ attention
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
// two probabilities of a word, times a factor
template <bool F16>
__device__ __forceinline__ uint32_t sh_scale(uint32_t w, float f) {
  if constexpr (F16) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return sh_pack<true>(v.x * f, v.y * f);
  } else {
    return sh_pack<false>(__uint_as_float(w << 16) * f, __uint_as_float(w & 0xFFFF0000u) * f);
  }
}
// V as the B operand: keys x head_dim with the head dimension contiguous (MN-major, 128-byte swizzle; see attention_tc.cu)
__device__ __forceinline__ uint64_t sh_desc_v(uint32_t smem_addr, uint32_t box) {
  return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(box >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

// One poll.  (mbar_wait's loop in line at every wait was half of the kernel's code, and the five programs of two CTAs outgrew the instruction cache.)
__device__ __forceinline__ bool mbar_test_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __noinline__ bool sh_wait_long(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int site) {
#pragma unroll 1
  for (int i = 0; i < 64; ++i)
    if (mbar_try_wait(bar, parity)) return true;
  return mbar_wait(bar, parity, abort_flag, status, site);
}
__device__ __forceinline__ bool sh_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status, int site) {
  return mbar_try_wait(bar, parity) || sh_wait_long(bar, parity, abort_flag, status, site);
}

struct ShArgs {
  const int *row_seq, *ctx_len, *common;      // of a window that the kernel plans, to `planned`; else nullptr
  int* planned;
  const int* block_table;
  const int* plan;
  const float* kv_scale;
  float* part_o;
  float* part_ml;
  int* status;
  int max_blocks, n_q, n_kv, rows, n_tables;
  float scale_log2;
};

template <int HD, bool F8>
struct Sh {
  static constexpr int TILE = SH_PAGE * HD * 2, QBOX = SH_PAIRS * 128;      // a page of K or V as an operand; 64 values of all pairs
  static constexpr int RAW = SH_PAGE * HD, RS = F8 ? 2 : 0;                 // a byte page; stages of those, of K and of V each
  static constexpr int KS = F8 ? 1 : 3, VS = 2;                             // stages of operand pages of K, of V
  static constexpr int KC = F8 ? RS : KS, VC = F8 ? RS : VS, COPY = F8 ? RAW : TILE;      // what the copies fill
  static constexpr int SMEM = (KS + VS) * TILE + 2 * RS * RAW + HD / 64 * QBOX + 1024;    // two CTAs an SM: 115,712 bytes at most
  static_assert(SMEM <= 115712, "two CTAs an SM");
  static constexpr int THREADS = 32 * (F8 ? 10 : 6);
  // fp16 has no values below 2^-24 and few below 2^-14: its operands are the probabilities times 2^7 (at most 2^15), so that what is lost of a key is at most 2^-32 of the
  // row's largest.  (As they are, 2^-25: 30,000 keys of that size, in the row's sum but not in its outputs, were a thousandth of it.)
  static constexpr float UP = F8 ? 7.f : 0.f;
  static constexpr int S_COLS = 64, O = 128, COLS = 256;                    // tensor memory: two buffers of S (P over the first 32 columns of one) | O
};

// a wait's outcome for the whole warp: what follows it is done by all lanes or by none
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok); }

// The CTA's piece of the line as segments: its pages of one unit each.
struct ShSegment { int row, rows, slots, seq, kvh, page, pages, slot, part, most; };
struct ShWalk {
  const int4* blk;
  int4 x, y, nx, ny;                                                        // the block and the one behind it, on its way
  int b, last, kvh, pos, end, n_kv, L;
  __device__ __forceinline__ void fetch() {
    const int at = min(b + 1, last) * 2;
    nx = blk[at], ny = blk[at + 1];
  }
  __device__ __forceinline__ ShWalk(const int* plan, int n_kv_, bool fits) : n_kv(n_kv_) {
    const int all = plan[0], total = fits ? all : 0;
    L = plan[1], last = plan[2] - 1;
    b = plan[SH_HEAD + blockIdx.x];
    blk = reinterpret_cast<const int4*>(plan + SH_AT_BLOCKS);
    pos = (int)min((long long)total, (long long)blockIdx.x * L), end = (int)min((long long)total, (long long)pos + L);
    if (pos >= end) return;
    x = blk[2 * b], y = blk[2 * b + 1];
    fetch();
    kvh = (pos - y.y * n_kv) / (y.x + SH_SEGMENT);                          // (the plan gives the block that holds the piece's begin)
  }
  __device__ __forceinline__ bool next(ShSegment& s) {
    while (pos < end) {
      const int len = y.x + SH_SEGMENT, unit = y.y * n_kv + kvh * len + SH_SEGMENT, stop = min(end, unit + y.x);
      s.page = max(pos - unit, 0), s.pages = stop - max(pos, unit);
      // a unit that begins in this piece meets this CTA first
      s.slot = s.page > 0 ? (int)blockIdx.x - unit / L : 0;
      s.row = x.x, s.rows = x.y & 255, s.slots = x.y >> 8, s.seq = x.z, s.page += x.w, s.kvh = kvh, s.part = y.z, s.most = y.w;
      pos = unit + y.x;
      if (++kvh == n_kv) {
        kvh = 0, ++b;
        x = nx, y = ny;
        fetch();
      }
      if (s.pages > 0) return true;                                         // (else the piece ended before the unit's first page)
    }
    return false;
  }
};

// What the warps know of a segment; the eight last are in shared memory.  pages == 0: there are no more.
struct alignas(16) ShDesc {
  int row, rows, kvh, key0, pages, part, stride, most;
  const int* table;       // its page ids
};

// N columns of the thread's lane, once they are there (load and wait in one statement: no copy of a register comes between them)
template <int N>
__device__ __forceinline__ void sh_ld(uint32_t taddr, uint32_t (&r)[N]) {
  static_assert(N == 64 || N == 32 || N == 16 || N == 8, "8, 16, 32 or 64 columns");
  if constexpr (N == 64)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
                 "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, "
                 "%46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                   "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]),
                   "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]),
                   "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),
                   "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
                 : "r"(taddr)
                 : "memory");
  else if constexpr (N == 32)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, "
                 "%20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
                   "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(taddr)
                 : "memory");
  else if constexpr (N == 8)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
  else if constexpr (N == 16)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
                 "[%16];\n\ttcgen05.wait::ld.sync.aligned;"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                   "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
// 32 columns of 16 lanes: thread t has columns 8 k + 2 (t % 4) and the next of lane t / 4 in r[4 k], r[4 k + 1] and of lane t / 4 + 8 in r[4 k + 2], r[4 k + 3]
__device__ __forceinline__ void sh_ld_16x256b_x4(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
                 "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
               : "r"(taddr)
               : "memory");
}
template <int N>
__device__ __forceinline__ void sh_st(uint32_t taddr, const uint32_t (&r)[N]) {
  static_assert(N == 32 || N == 16 || N == 8, "8, 16 or 32 columns");
  if constexpr (N == 32) tc_st_32x32b_x32(taddr, r);
  else if constexpr (N == 16) tc_st_32x32b_x16(taddr, r);
  else if constexpr (N == 8)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
template <int N>
__device__ __forceinline__ void sh_st_zero(uint32_t taddr) {
  const uint32_t z[N] = {};
  sh_st(taddr, z);
}

// The query heads of a KV head, 64 of their values each, from [rows][n_q][hd]: of as many rows at once as fill a quarter of the pairs
__host__ __device__ constexpr int sh_box_rows(int G) { return G > 32 ? 1 : 32 / G; }
__device__ __forceinline__ void sh_load_q(void* dst, const void* tmap, int x, int head, int row, uint64_t* bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)), "l"(tmap),
               "r"(smem_u32(bar)), "r"(x), "r"(head), "r"(row)
               : "memory");
}

// the rows of a V page from `first` on, by the four softmax warps
__device__ __noinline__ bool sh_zero_rows(uint8_t* page, int boxes, int first) {
  for (int x = 0; x < boxes; ++x)
    for (int i = first * 8 + (int)threadIdx.x; i < SH_PAGE * 8; i += 128) *reinterpret_cast<uint4*>(page + x * 8192 + i * 16) = make_uint4(0u, 0u, 0u, 0u);
  fence_proxy_async();
  return true;
}

template <int HD, bool F8>
__global__ void __launch_bounds__((Sh<HD, F8>::THREADS), 2)
attn_shared_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tq, const __grid_constant__ ShArgs a) {
  using C = Sh<HD, F8>;
  constexpr int BOXES = HD / 64, TILE = C::TILE, KS = C::KS, VS = C::VS;
  pdl_launch();
  extern __shared__ __align__(1024) uint8_t smem[];
  if ((smem_u32(smem) & 1023) != 0) {                     // (a kernel without static shared memory begins on a 1024-byte boundary)
    if (threadIdx.x == 0) set_status(a.status, ST_BAD_ARG, 109);
    return;
  }
  uint8_t* k_sm = smem;                                   // [stage][box (64 d)][64 keys][128 B]
  uint8_t* v_sm = smem + KS * TILE;
  uint8_t* q_sm = smem + (KS + VS) * TILE;                // [box][128 pairs][128 B]
  uint8_t* raw = q_sm + BOXES * C::QBOX;                  // [K, V][stage][64 keys][HD]
  uint64_t* bars = (uint64_t*)(raw + 2 * C::RS * C::RAW);
  uint64_t* k_full = bars;                                // [KS] the copies, or the two expanding warps
  uint64_t* v_full = k_full + KS;                         // [VS]
  uint64_t* raw_empty = v_full + VS;                      // [K, V][RS] the two expanding warps
  uint64_t* raw_full = raw_empty + 2 * C::RS;             // [K, V][RS] the copy
  uint64_t* k_empty = raw_full + 2 * C::RS;               // [KS] commit after QK
  uint64_t* v_empty = k_empty + KS;                       // [VS] commit after PV
  uint64_t* s_full = v_empty + VS;                        // [2] commit after QK
  uint64_t* pv_done = s_full + 2;                         // [2] commit after PV
  uint64_t* q_ready = pv_done + 2;                        // [4] a segment's queries and description are there
  uint64_t* q_free = q_ready + 4;                         // commit after a segment's last QK
  uint64_t* drained = q_free + 1;
  uint64_t* q_there = drained + 1;                        // (E4M3 caches) the queries as they are
  uint64_t* p_ready = q_there + 1;                        // [2] the 4 softmax warps
  ShDesc* desc = (ShDesc*)(((uintptr_t)(p_ready + 2) + 15) & ~(uintptr_t)15);      // [8]
  uint32_t* tmem_slot = (uint32_t*)(desc + 8);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* pages_all = abort_flag + 1;               // (E4M3 caches) pages of the CTA's piece, once the last has been asked for
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (uint64_t* bar = bars; bar < p_ready; ++bar) mbar_init(bar, F8 && bar < raw_full ? 2 : 1);      // (two expanding warps)
    mbar_init(&p_ready[0], 4);
    mbar_init(&p_ready[1], 4);
    *abort_flag = 0;
    *pages_all = 0x7FFFFFFF;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, C::COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();                                             // the plan, q and the caches were written by the previous kernels
  const uint32_t tmem_base = *tmem_slot;
  const int G = a.n_q / a.n_kv;
  if (a.row_seq != nullptr)
    sh_plan_here(smem, a.row_seq, a.ctx_len, a.common, a.rows, a.n_tables, a.max_blocks, G, a.n_kv, a.planned, a.status);

  if (warp < 4) {
    // ---------------------------------------------------------------- softmax warps: thread = (row, head) pair or a copy of it = TMEM lane
    const uint32_t lane_addr = tmem_base + ((uint32_t)(warp * 32) << 16);
    int n = 0;                                            // pages so far
    bool ok = true;
    for (int seg = 0; ok; ++seg) {
      ok = all_ok(sh_wait(&q_ready[seg & 3], (seg >> 2) & 1, abort_flag, a.status, 110));
      if (!ok) break;
      const ShDesc d = desc[seg & 7];
      if (d.pages == 0) break;
      const int pairs = d.rows * G, copies = sh_copies(pairs);
      const int copy = copies == 4 ? warp : copies == 2 ? warp >> 1 : 0, pair = copies == 4 ? lane : copies == 2 ? (warp & 1) * 32 + lane : warp * 32 + lane;
      const int rb = pair / G, hq = d.kvh * G + pair % G;
      const bool live = rb < d.rows, some = copies > 1 || warp * 32 < pairs;         // (uniform) the warp holds a pair
      // keys from the segment's first on that the pair sees (a lane without a pair: nothing to mask, nothing comes of it)
      const int keys = live ? a.plan[SH_AT_KEYS + d.row + rb] - d.key0 : 0x7FFFFFFF;
      const float scale_log2 = F8 ? a.scale_log2 * a.kv_scale[d.kvh] : a.scale_log2;
      float m = -INFINITY, l = 0.f;                       // running maximum (log2 units), sum
      // Keys that no row sees yet: their V may hold anything, and 0 * NaN would reach every pair.  (The barrier of V's stage cannot stand a page's use behind: that
      // PV was over before the scores of this page were.)
      auto tail = [&](int j) {
        const int first = max(d.most - d.key0 - j * SH_PAGE, 0);
        return first >= SH_PAGE || (all_ok(sh_wait(&v_full[n % VS], (n / VS) & 1, abort_flag, a.status, 104)) && sh_zero_rows(v_sm + (n % VS) * TILE, BOXES, first));
      };
      // The segment's pages, NC columns a thread at a time: `parts` times for the 64 / copies scores of a page that are the thread's.  (The code is kept small: the
      // warps of two CTAs run five programs at once, and where those outgrew the instruction cache, warps waited for it five cycles an instruction.)
      auto pages = [&](auto nc, int parts) {
        constexpr int NC = decltype(nc)::value;
        const int col = NC * parts * copy;
        uint32_t s[NC];
        auto scores = [&](int at, int part) {             // of the CTA's page `at`
          tc_fence_after();
          sh_ld(lane_addr + (at & 1) * C::S_COLS + col + part * NC, s);
        };
        // scores -> probabilities, over the first half of the columns: those have been read
        auto exponentials = [&](int j, int part) {
          int seen = keys == 0x7FFFFFFF ? NC : keys - j * SH_PAGE - col - part * NC;
          asm volatile("" : "+r"(seen));                  // (else the bounds of all columns are held in registers over the whole segment)
          if (seen < NC) {
#pragma unroll
            for (int i = 0; i < NC; ++i)
              if (i >= seen) s[i] = 0xFF800000u;
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < NC; ++i) mx[i & 3] = fmaxf(mx[i & 3], __uint_as_float(s[i]));
          const float ms = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale_log2;
          // The running maximum moves only by more than 2^8: the probabilities stay below 2^8 (2^15 with UP), harmless in 16-bit operands and fp32 sums.  (A move in a page's second
          // part comes before the first part's product: those probabilities would be of the old maximum.  So they move with O.)
          const bool moves = live && ms > m + 8.f;        // (a lane without a pair has another's old queries, or none: its scores may be anything)
          if (__any_sync(0xffffffffu, moves)) {           // all pages but a segment's first few: no
            float alpha = 1.f;
            if (moves) {
              if (m != -INFINITY) alpha = sh_ex2(m - ms);
              m = ms;
            }
            l *= alpha;
            if (__any_sync(0xffffffffu, alpha != 1.f)) {
              if (part > 0) {                             // this page's first probabilities
                tc_wait_st();
#pragma unroll 1
                for (int p = 0; p < part; ++p) {
                  uint32_t r[NC / 2];
                  const uint32_t at = lane_addr + (n & 1) * C::S_COLS + (col + p * NC) / 2;
                  sh_ld(at, r);
#pragma unroll
                  for (int i = 0; i < NC / 2; ++i) r[i] = sh_scale<F8>(r[i], alpha);
                  sh_st(at, r);
                }
              }
              if (j > 0) {                                // O, as the PV before leaves it
                if (!all_ok(sh_wait(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, a.status, 103))) return false;
                tc_fence_after();
#pragma unroll 1
                for (int ch = 0; ch < HD / 16; ++ch) {
                  uint32_t r[16];
                  sh_ld(lane_addr + C::O + ch * 16, r);
#pragma unroll
                  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                  sh_st(lane_addr + C::O + ch * 16, r);
                }
              }
            }
          }
          const float m_use = (m == -INFINITY) ? 0.f : m - Sh<HD, F8>::UP;      // (sum and outputs are 2^UP times as large alike: nothing is to be undone)
          float lsum[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t pk[NC / 2];
#pragma unroll
          for (int i = 0; i < NC / 2; ++i) {
            const float pa = sh_ex2(fmaf(__uint_as_float(s[2 * i]), scale_log2, -m_use)), pb = sh_ex2(fmaf(__uint_as_float(s[2 * i + 1]), scale_log2, -m_use));
            lsum[i & 3] += pa + pb;
            pk[i] = sh_pack<F8>(pa, pb);
          }
          l += (lsum[0] + lsum[1]) + (lsum[2] + lsum[3]);
          sh_st(lane_addr + (n & 1) * C::S_COLS + (col + part * NC) / 2, pk);
          return true;
        };
        if (!all_ok(sh_wait(&s_full[n & 1], (n >> 1) & 1, abort_flag, a.status, 102))) return false;
        scores(n, 0);
        for (int j = 0;; ++j, ++n) {
#pragma unroll 1
          for (int part = 0;;) {
            if (!exponentials(j, part)) return false;
            if (++part == parts) break;
            scores(n, part);
          }
          // the other copies' columns of P
          const uint32_t s_addr = lane_addr + (n & 1) * C::S_COLS;
          if (copies == 2) sh_st_zero<16>(s_addr + 16 * (1 - copy));
          if (copies == 4) {
#pragma unroll
            for (int o = 1; o < 4; ++o) sh_st_zero<8>(s_addr + 8 * ((copy + o) & 3));
          }
          // The next page's scores are fetched while the probabilities are on their way, if they are there: where a page's exponentials are quickly done, waiting for
          // them (they come after the PV before) would be what takes longest.
          const bool last = j + 1 == d.pages;
          const bool early = !last && all_ok(mbar_test_wait(&s_full[(n + 1) & 1], ((n + 1) >> 1) & 1));
          if (early) scores(n + 1, 0);
          tc_wait_st();
          tc_fence_before();
          if (!tail(j)) return false;
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_ready[n & 1]);
          if (last) {
            ++n;
            return true;
          }
          if (!early) {
            if (!all_ok(sh_wait(&s_full[(n + 1) & 1], ((n + 1) >> 1) & 1, abort_flag, a.status, 102))) return false;
            scores(n + 1, 0);
          }
        }
      };
      if (!some) {
        for (int j = 0; j < d.pages && ok; ++j, ++n) {
          ok = all_ok(sh_wait(&s_full[n & 1], (n >> 1) & 1, abort_flag, a.status, 102)) && tail(j);
          __syncwarp();                                   // (the tail's zeros are all lanes')
          if (ok && lane == 0) mbar_arrive(&p_ready[n & 1]);
        }
      } else {
        // 64 / copies = NC * parts
        if constexpr (F8) ok = copies == 4 ? pages(std::integral_constant<int, 16>(), 1) : pages(std::integral_constant<int, 32>(), 2 / copies);
        else ok = copies == 1 ? pages(std::integral_constant<int, 64>(), 1) : pages(std::integral_constant<int, 16>(), 4 / copies);
      }
      if (ok) ok = all_ok(sh_wait(&pv_done[(n - 1) & 1], ((n - 1) >> 1) & 1, abort_flag, a.status, 105));
      if (ok && some) {
        tc_fence_after();
        const float v_scale = F8 ? a.kv_scale[a.n_kv + d.kvh] : 1.f;
        const int at = live ? (d.part + rb * d.stride + copy) * a.n_q + hq : -1;
        if (live) *reinterpret_cast<float2*>(a.part_ml + (size_t)at * 2) = make_float2(m, l);
        // Eight lanes' rows by four lanes each: two neighbouring lanes swap pairs, so that a store writes 64 bytes of each of eight rows.  (A row by its own thread, 32
        // rows a store, took 6300 cycles a segment.)
#pragma unroll 1
        for (int ch = 0; ch < HD / 16; ++ch) {
          const int cols = ch >> 1, h = ch & 1;           // 32 columns of the upper or lower 16 rows
          uint32_t r[16];
          sh_ld_16x256b_x4(lane_addr + ((uint32_t)(h * 16) << 16) + C::O + cols * 32, r);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int row = __shfl_sync(0xffffffffu, at, h * 16 + u * 8 + (lane >> 2));
#pragma unroll
            for (int k = 0; k < 2; ++k) {                 // r[8 k + 2 u ..]: columns 16 k + 2 (lane % 4) ..; r[8 k + 4 + 2 u ..]: eight further
              const uint32_t a0 = r[8 * k + 2 * u], a1 = r[8 * k + 2 * u + 1], b0 = r[8 * k + 4 + 2 * u], b1 = r[8 * k + 5 + 2 * u];
              const bool odd = lane & 1;
              const uint32_t g0 = __shfl_xor_sync(0xffffffffu, odd ? a0 : b0, 1), g1 = __shfl_xor_sync(0xffffffffu, odd ? a1 : b1, 1);
              if (row >= 0)
                *reinterpret_cast<float4*>(a.part_o + (size_t)row * HD + cols * 32 + k * 16 + (odd ? 8 : 0) + (lane & 2) * 2) =
                    make_float4(__uint_as_float(odd ? g0 : a0) * v_scale, __uint_as_float(odd ? g1 : a1) * v_scale, __uint_as_float(odd ? b0 : g0) * v_scale,
                                __uint_as_float(odd ? b1 : g1) * v_scale);
            }
          }
        }
        tc_fence_before();                                // the reads of O are ordered before the next segment's first PV by p_ready
      }
    }
  } else if (warp == 4) {
    // ---------------------------------------------------------------- feeder: descriptions and queries of the segments; K and V each at their own pace
    // One warp's ordinary code is slow (some five cycles an instruction), so it does little of it: a segment is looked up once for everybody, and its
    // queries come by TMA, several rows' heads of one KV head per copy (by plain copies, 125 pairs took 25,000 cycles, by a copy a row 5000).
    // (With K and V in turn, K page n + 2 waited for V page n + 1 and so for PV(n - 1), and a page took as long as a K page's way from memory.)
    // Of eight descriptions the one that is overwritten, segment w - 8's, is out of use: V has begun segment w - 1, with a page whose copy waited for the PV of a page
    // two (E4M3: four) earlier, in segment w - 5 or later, and that PV for all softmax warps to leave the segments before.
    const bool fits = sh_fits(a.plan, a.n_kv, a.n_q, a.rows, a.n_tables, a.max_blocks);      // (else there is nothing to do, and the merge gives zeros)
    if (!fits && blockIdx.x == 0 && lane == 0) set_status(a.status, ST_BAD_ARG, 97, a.plan[5]);
    ShWalk walk(a.plan, a.n_kv, fits);
    int known = 0, asked = 0, queries = 0, converted = 0, idle = 0;      // segments with a description, with queries; the last one whose queries were fetched, + 1
    bool more = true;
    uint64_t since = 0;
    // lane 0 brings K, lane 1 V: the ring's place, and the pages that are left of the lane's segment
    const int S = lane == 0 ? C::KC : C::VC, who = lane & 1;
    uint64_t *full = F8 ? raw_full + who * C::RS : who ? v_full : k_full, *empty = F8 ? raw_empty + who * C::RS : who ? v_empty : k_empty;
    uint8_t* to = F8 ? raw + who * C::RS * C::RAW : who ? v_sm : k_sm;
    const CUtensorMap* map = who ? &tv : &tk;
    const unsigned pages_end = (1u << 31) / SH_PAGE / a.n_kv;      // page ids whose rows int32 can count
    const int* table = nullptr;                            // of the lane's segment, behind the page that comes next: that one is known before its place is free
    int at = 0, next = 0, begun = 0, st = 0, round = 0, left = 0, kvh = 0, copied = 0;      // segments looked at, and begun; the ring's place; pages left of the segment, asked for
    bool done = lane > 1;
    while (more || asked < known || (F8 && converted < queries) || __any_sync(0xffffffffu, !done)) {
      bool moved = false;
      if (asked < known && (asked == 0 || all_ok(mbar_test_wait(q_free, (asked - 1) & 1)))) {
        const ShDesc& d = desc[asked & 7];
        // (the last box of several begins early enough to end with the block; one alone may reach rows behind it, which nothing comes of)
        const int rows = d.pages != 0 ? d.rows : 0, copies = sh_copies(rows * G), most = sh_box_rows(G), boxes = (rows + most - 1) / most;
        const int bytes = boxes * most * copies * G * HD * 2;
        uint64_t* bar = F8 ? q_there : &q_ready[asked & 3];
        if (lane == 0) {
          if (bytes != 0) mbar_arrive_expect_tx(bar, bytes);
          else mbar_arrive(&q_ready[asked & 3]);
        }
        __syncwarp();
        // 128-byte rows at any multiple of 128 bytes: the swizzle goes by the address, so chunk c of pair p stands at c ^ (p & 7)
        for (int i = lane; i < boxes * copies * BOXES; i += 32) {
          const int x = i % BOXES, t = i / BOXES & (copies - 1), b = i / BOXES >> (copies >> 1), r = b + 1 < boxes || b == 0 ? b * most : rows - most;
          sh_load_q(q_sm + x * C::QBOX + (t * (SH_PAIRS / copies) + r * G) * 128, &tq, x * 64, d.kvh * G, d.row + r, bar);
        }
        __syncwarp();
        if (rows != 0) queries = asked + 1;
        ++asked;
        moved = true;
      }
      if (!done) {
        if (left == 0 && at < known) {
          const ShDesc& d = desc[at & 7];
          left = d.pages, table = d.table, kvh = d.kvh;
          done = left == 0;
          if (!done) next = *table++;
          ++at;
        }
        if (left != 0 && (round == 0 || mbar_test_wait(&empty[st], (round - 1) & 1))) {
          const int y = (unsigned)next < pages_end ? (next * a.n_kv + kvh) * SH_PAGE : -SH_PAGE;      // (outside the cache: zeros)
          mbar_arrive_expect_tx(&full[st], C::COPY);
#pragma unroll
          for (int x = 0; x < (F8 ? 1 : BOXES); ++x) tma_load_2d(to + st * C::COPY + x * 8192, map, x * 64, y, &full[st]);
          if (--left != 0) next = *table++;
          ++copied;
          begun = at;
          if (++st == S) st = 0, ++round;
          moved = true;
        }
      }
      __syncwarp();
      if (F8 && converted < queries && all_ok(mbar_test_wait(q_there, converted & 1))) {      // bf16 -> fp16 in place, beside the fp16 values of an E4M3 cache
        const int rows = desc[converted & 7].rows, copies = sh_copies(rows * G);
        for (int t = 0; t < copies; ++t)
#pragma unroll
          for (int x = 0; x < BOXES; ++x) {
            const uint32_t at = smem_u32(q_sm + x * C::QBOX + t * (SH_PAIRS / copies) * 128);
#pragma unroll 4
            for (int i = lane; i < rows * G * 8; i += 32) {
              uint4 v = lds128(at + i * 16);
              uint32_t* w = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
              for (int u = 0; u < 4; ++u) w[u] = sh_pack<true>(__uint_as_float(w[u] << 16), __uint_as_float(w[u] & 0xFFFF0000u));
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at + i * 16), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
            }
          }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[converted & 3]);
        ++converted;
        moved = true;
      }
      if (more && (known < 8 || __shfl_sync(0xffffffffu, begun, 1) >= known)) {
        ShSegment sg = {};
        more = walk.next(sg);
        const int copies = sh_copies(sg.rows * G);
        if (lane == 0)
          desc[known & 7] = ShDesc{sg.row, sg.rows, sg.kvh, sg.page * SH_PAGE, more ? sg.pages : 0, sg.part + sg.slot * copies, sg.slots * copies, sg.most,
                                   a.block_table + (size_t)sg.seq * a.max_blocks + sg.page};
        __syncwarp();
        ++known;
        moved = true;
      }
      if (__any_sync(0xffffffffu, moved)) {
        idle = 0;
      } else if (++idle > 64) {
        __nanosleep(20);
        if ((idle & 511) == 0) {                          // (a bounded wait, as mbar_wait's, for whatever can go on first)
          if (idle == 512) since = globaltimer_ns();
          const bool stop = host_abort(a.status), late = globaltimer_ns() - since > wait_limit_ns(a.status);
          if (lane == 0 && (stop || late)) set_status(a.status, stop ? ST_ABORTED : ST_TIMEOUT, 96), *abort_flag = 1;
          __syncwarp();
          if (__any_sync(0xffffffffu, *abort_flag != 0)) break;
        }
      }
    }
    __syncwarp();
    if (lane < 2) {
      ring_landed(full, S, copied);
      if constexpr (F8) {                                 // the expanding warps learn that there are no more
        if (lane == 0) *pages_all = copied;
        __syncwarp(3);
        // (The place must be free, as for a copy: else the barrier could go on by two phases while a warp still waits for the first, of the page before last.)
        if (round == 0 || sh_wait(&empty[st], (round - 1) & 1, abort_flag, a.status, 111)) mbar_arrive(&full[st]);
      }
    }
    if (lane == 0) {
      // (where the others gave up, nobody has waited for the last queries)
      uint64_t* last = F8 ? q_there : &q_ready[(queries - 1) & 3];
      const int parity = (F8 ? queries - 1 : (queries - 1) >> 2) & 1;
      if (*abort_flag != 0 && queries > 0)
        for (int i = 0; i < (1 << 20) && !mbar_try_wait(last, parity); ++i) __nanosleep(100);
    }
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA issuer
    if (elect_one()) {
      constexpr uint32_t fmt = F8 ? 0 : 1;
      constexpr uint32_t idesc_qk = umma_idesc_f16(SH_PAIRS, SH_PAGE, fmt, fmt);              // both K-major
      constexpr uint32_t idesc_pv = umma_idesc_f16(SH_PAIRS, HD, fmt, fmt) | (1u << 16);      // B (V) is MN-major
      const uint64_t qd = umma_desc_k_sw128(smem_u32(q_sm));
      // Whatever can go on first goes: the next page's QK, up to two pages ahead of the PVs and into the next segment, or the next PV.  (In a fixed order, the PV of a
      // segment's last page stood behind the next segment's queries.)
      int n = 0, p = 0, seg_qk = 0, left_qk = 0, seg = 0, left = 0, idle = 0;      // pages with a QK, with a PV; segments begun and pages left of the segment, of each
      bool more = true;
      uint64_t since = 0;
#pragma unroll 1
      while (more || p < n) {
        if (more && n - p < 2) {
          if (left_qk == 0 && mbar_test_wait(&q_ready[seg_qk & 3], (seg_qk >> 2) & 1)) {
            left_qk = desc[seg_qk & 7].pages;
            if (left_qk == 0) {
              more = false;
              continue;
            }
            ++seg_qk;
          }
          const int st = n % KS;
          if (left_qk != 0 && mbar_test_wait(&k_full[st], (n / KS) & 1)) {
            tc_fence_after();
            const uint64_t kd = umma_desc_k_sw128(smem_u32(k_sm + st * TILE));
#pragma unroll
            for (int kk = 0; kk < HD / 16; ++kk)
              tc_mma_f16(tmem_base + (n & 1) * C::S_COLS, qd + (uint64_t)((kk >> 2) * (C::QBOX >> 4) + (kk & 3) * 2), kd + (uint64_t)((kk >> 2) * (8192 >> 4) + (kk & 3) * 2),
                         idesc_qk, kk != 0);
            tc_commit(&s_full[n & 1]);                    // (over P(n - 2), which its PV has read: a thread's MMAs run in issue order)
            tc_commit(&k_empty[st]);
            if (--left_qk == 0) tc_commit(q_free);
            ++n;
            idle = 0;
            continue;
          }
        }
        const int st = p % VS;
        if (p < n && mbar_test_wait(&p_ready[p & 1], (p >> 1) & 1) && mbar_test_wait(&v_full[st], (p / VS) & 1)) {
          const bool fresh = left == 0;
          if (fresh) left = desc[seg++ & 7].pages;
          --left;
          tc_fence_after();
          const uint64_t vd = sh_desc_v(smem_u32(v_sm + st * TILE), 8192);
#pragma unroll
          for (int kk = 0; kk < SH_PAGE / 16; ++kk)
            tc_mma_f16_ts(tmem_base + C::O, tmem_base + (p & 1) * C::S_COLS + kk * 8, vd + (uint64_t)(kk * (2048 >> 4)), idesc_pv, !fresh || kk != 0);
          tc_commit(&pv_done[p & 1]);
          tc_commit(&v_empty[st]);
          ++p;
          idle = 0;
          continue;
        }
        if ((++idle & 4095) == 0) {                       // (bounded, as mbar_wait is)
          if (idle == 4096) since = globaltimer_ns();
          const bool stop = host_abort(a.status), late = globaltimer_ns() - since > wait_limit_ns(a.status);
          if (stop || late) set_status(a.status, stop ? ST_ABORTED : ST_TIMEOUT, 98, n), *abort_flag = 1;
          if (*abort_flag != 0) break;
        }
      }
      // every MMA issued so far has completed when this commit arrives: the columns may then be returned
      tc_commit(drained);
      for (int i = 0; i < (1 << 22) && !mbar_try_wait(drained, 0); ++i) {}   // bounded, and not cut short by the abort word
    }
  } else if constexpr (F8) {
    // ---------------------------------------------------------------- expansion of byte pages: E4M3 -> fp16 (exact) in the operand layout
    // A warp takes half of every page of K or of V.  (Straight from global memory, a page ahead in registers, a page took 3300 cycles: the way of plain loads.)
    // Eight lanes take two keys, of 128-byte rows a half each: neither loads nor stores then meet in a bank.
    const int v = (warp - 6) >> 1, half = warp & 1, S = v ? VS : KS;
    uint64_t *full = v ? v_full : k_full, *empty = v ? v_empty : k_empty, *rfull = raw_full + v * C::RS, *rempty = raw_empty + v * C::RS;
    // (bytes) lane's first 16 values of a page, of even and - rows of 128 bytes - odd turns; where they go, in two chunks; from turn to turn (pair of turns to pair) both
    // move by whole groups of eight keys
    constexpr int TURNS = HD / 16, ODD = HD == 128 ? 2 : 1;
    const int key = half * 32 + (HD == 128 ? (lane >> 3) * 2 + (lane >> 2 & 1) : lane >> 2);
    uint32_t from[ODD], into[ODD][2];
#pragma unroll
    for (int o = 0; o < ODD; ++o) {
      const int x = (lane & 3) + (HD == 128 ? 4 * ((lane >> 2 & 1) ^ o) : 0);
      from[o] = key * HD + x * 16;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int ch = 2 * x + u;                         // 16-byte chunk of the fp16 row
        into[o][u] = (ch >> 3) * 8192 + key * 128 + (((ch & 7) ^ (key & 7)) << 4);
      }
    }
    for (int n = 0;; ++n) {
      const int rs = n % C::RS, st = n % S;
      if (!all_ok(sh_wait(&rfull[rs], (n / C::RS) & 1, abort_flag, a.status, 106)) || n >= *pages_all) break;
      const uint32_t src = smem_u32(raw + (v * C::RS + rs) * C::RAW), dst = smem_u32((v ? v_sm : k_sm) + st * TILE);
      uint4 b[TURNS];
#pragma unroll
      for (int i = 0; i < TURNS; ++i) b[i] = lds128(src + from[i % ODD] + i / ODD * 8 * HD);
      if (n >= S && !all_ok(sh_wait(&empty[st], ((n / S) - 1) & 1, abort_flag, a.status, 107))) break;
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const uint32_t w[4] = {b[i].x, b[i].y, b[i].z, b[i].w};
        uint32_t e[8];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, l;\n\tcvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(e[2 * u]), "=r"(e[2 * u + 1]) : "r"(w[u]));
#pragma unroll
        for (int u = 0; u < 2; ++u)
          asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + into[i % ODD][u] + i / ODD * 1024), "r"(e[4 * u]), "r"(e[4 * u + 1]), "r"(e[4 * u + 2]),
                       "r"(e[4 * u + 3])
                       : "memory");
      }
      fence_proxy_async();
      __syncwarp();
      // (the bytes' place is given back only here: an arrival does not wait for loads whose values nothing has used yet)
      if (lane == 0) {
        mbar_arrive(&full[st]);
        mbar_arrive(&rempty[rs]);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 5) tmem_dealloc(tmem_base, C::COLS);
}

// ------------------------------------------------------------------------------------------------ merge
// Joins a row's partial outputs, common pages before own, CTA by CTA: out = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  128 outputs by SPLIT warps, each
// with every SPLIT-th slot, and U partial outputs of a warp on their way at once; with `suh` also xr = fp16(H(out * suh)), the input rotation of the output projection.
template <int HD, int SPLIT, int U>
__global__ void __launch_bounds__(SPLIT > 4 ? 32 * SPLIT : 128) attn_shared_merge_kernel(const int* plan, const float* part_o, const float* part_ml, int n_q, int n_kv,
                                                                                         int n_tables, int max_blocks, const __half* __restrict__ suh,
                                                                                         __half* __restrict__ xr, uint16_t* __restrict__ out) {
  pdl_launch();
  __shared__ float4 s_acc[SPLIT][32];
  __shared__ float2 s_ml[SPLIT][32];
  const int row = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, width = n_q * HD, who = SPLIT > 1 ? warp : 0;
  const int b = SPLIT > 1 ? blockIdx.y : blockIdx.y * 4 + warp, e0 = b * 128 + lane * 4, hq = e0 / HD, d0 = e0 % HD, kvh = hq / (n_q / n_kv);
  pdl_wait();
  if (b >= width / 128) return;                           // (a whole warp; with SPLIT none)
  const bool fits = sh_fits(plan, n_kv, n_q, gridDim.x, n_tables, max_blocks);
  const int L = plan[1];
  const int4* of = reinterpret_cast<const int4*>(plan + SH_AT_ROWS) + 2 * row;
  size_t at[2] = {0, 0};
  int n[2] = {0, 0};
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int4 s = of[u];                                  // before, pages, partial vectors, copies
    if (s.y == 0 || !fits) continue;
    const int unit = sh_unit(s.x, s.y, kvh, n_kv);
    n[u] = ((unit + s.y - 1) / L - unit / L + 1) * s.w;
    at[u] = (size_t)s.z * n_q + hq;
  }
  auto slot = [&](int i) {
    const int s = i * SPLIT + who;
    return s < n[0] ? at[0] + (size_t)s * n_q : at[1] + (size_t)(s - n[0]) * n_q;
  };
  const int all = (n[0] + n[1] - who + SPLIT - 1) / SPLIT;      // the warp's slots
  // A head's GL lanes take GL slots at a time, lane = slot for the maxima and factors.  (Two heads of 64 in a warp may have unlike numbers of slots.)
  constexpr int GL = HD / 4;
  static_assert(GL % U == 0, "whole turns");
  const int gl = lane % GL, g0 = lane - gl, most = HD == 128 ? all : max(all, __shfl_xor_sync(0xffffffffu, all, 16));
  float acc[4] = {0.f, 0.f, 0.f, 0.f}, l = 0.f, m = -INFINITY;
  for (int s0 = 0; s0 < most; s0 += GL) {
    const int here = min(GL, all - s0);                   // (of the other head of the warp, maybe none)
    const float2 ml = gl < here ? *reinterpret_cast<const float2*>(part_ml + slot(s0 + gl) * 2) : make_float2(-INFINITY, 0.f);
    float4 o[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < here) o[u] = *reinterpret_cast<const float4*>(part_o + slot(s0 + u) * HD + d0);
    float top = ml.x;
#pragma unroll
    for (int w = GL / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    top = fmaxf(m, top);
    const float old = m == -INFINITY ? 0.f : exp2f(m - top), f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
    m = top;
    l = l * old + f * ml.y;                               // (lane = slot: added up at the end)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= old;
#pragma unroll
    for (int u0 = 0; u0 < GL; u0 += U) {
      if (u0 > 0) {
        if (u0 >= min(GL, most - s0)) break;
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (u0 + u < here) o[u] = *reinterpret_cast<const float4*>(part_o + slot(s0 + u0 + u) * HD + d0);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float g = __shfl_sync(0xffffffffu, f, g0 + u0 + u);
        if (u0 + u < here) acc[0] += g * o[u].x, acc[1] += g * o[u].y, acc[2] += g * o[u].z, acc[3] += g * o[u].w;
      }
    }
  }
#pragma unroll
  for (int w = GL / 2; w > 0; w >>= 1) l += __shfl_xor_sync(0xffffffffu, l, w);
  if constexpr (SPLIT > 1) {
    s_acc[who][lane] = make_float4(acc[0], acc[1], acc[2], acc[3]);
    s_ml[who][lane] = make_float2(m, l);
    __syncthreads();
    if (who != 0) return;
    float top = m;
#pragma unroll
    for (int w = 1; w < SPLIT; ++w) top = fmaxf(top, s_ml[w][lane].x);
    const float own = m == -INFINITY ? 0.f : exp2f(m - top);
    l *= own;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= own;
#pragma unroll 4
    for (int w = 1; w < SPLIT; ++w) {
      const float2 ml = s_ml[w][lane];
      const float4 o = s_acc[w][lane];
      const float f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - top);
      l += f * ml.y;
      acc[0] += f * o.x, acc[1] += f * o.y, acc[2] += f * o.z, acc[3] += f * o.w;
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) acc[i] = n[0] + n[1] > 0 ? acc[i] * inv : 0.f;
  if (out != nullptr) *reinterpret_cast<uint2*>(out + (size_t)row * width + e0) = make_uint2(sh_pack<false>(acc[0], acc[1]), sh_pack<false>(acc[2], acc[3]));
  if (xr != nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] *= __half2float(suh[e0 + i]);
    fwht128_warp(acc);
    *reinterpret_cast<uint2*>(xr + (size_t)row * width + e0) = make_uint2(sh_pack<true>(acc[0], acc[1]), sh_pack<true>(acc[2], acc[3]));
  }
}

template <int HD, bool F8>
static cudaError_t launch_shared(int dev, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& tq, const ShArgs& a, cudaStream_t st) {
  static bool configured[64];
  if (dev >= 64 || !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(attn_shared_kernel<HD, F8>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh<HD, F8>::SMEM);
    if (e != cudaSuccess) return e;
    if (dev < 64) configured[dev] = true;
  }
  return rx::launch(attn_shared_kernel<HD, F8>, dim3(SH_CTAS), dim3(Sh<HD, F8>::THREADS), Sh<HD, F8>::SMEM, st, tk, tv, tq, a);
}

// The queries [rows][n_q][hd] by boxes of some rows' G heads, 64 values of each.
static bool sh_query_map(CUtensorMap* map, const void* q, int rows, int n_q, int G, int hd) {
  typedef CUresult (*Encode)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                             CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static Encode encode = nullptr;
  if (encode == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) return false;
    encode = (Encode)p;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)n_q, (cuuint64_t)rows}, strides[2] = {(cuuint64_t)hd * 2, (cuuint64_t)n_q * hd * 2};
  const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)sh_box_rows(G)}, steps[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace rx

using namespace rx;

RX_API int rx_attn_shared_plan_ints() { return SH_PLAN_INTS; }

// Partial vectors: a unit meets at most pages / L + 2 CTAs, a block of n rows leaves n * copies from each, at most SH_PAIRS / G; all blocks' pages / L together
// are at most SH_CTAS / n_kv; a row is in two blocks, with up to four copies of it in each.
RX_API long long rx_attn_shared_scratch_floats(int rows, int n_q, int n_kv, int hd) {
  if (rows < 1 || n_q < 1 || n_kv < 1 || n_q % n_kv != 0 || n_q / n_kv > SH_PAIRS) return 0;
  const long long rt = SH_PAIRS / (n_q / n_kv), vectors = (rt * SH_CTAS / n_kv + 1 + 16ll * rows) * n_q;
  return vectors * (hd + 2) + SH_PLAN_INTS;
}

static bool sh_takes(int rows, int n_q, int n_kv, int n_tables, int max_blocks) {
  return rows >= 1 && rows <= SH_MAX_ROWS && n_kv >= 1 && n_q <= 65536 && n_q >= n_kv && n_q % n_kv == 0 && n_q / n_kv <= SH_PAIRS && n_tables >= 1 && max_blocks >= 1 &&
         (long long)rows * (max_blocks + SH_SEGMENT) * n_kv < (1ll << 29) && max_blocks < (1 << 24);
}

RX_API int rx_attn_shared_plan(const void* row_seq, const void* ctx_len, const void* common, int rows, int n_tables, int max_blocks, int n_q, int n_kv, void* plan,
                               int* status, void* stream) {
  if (!sh_takes(rows, n_q, n_kv, n_tables, max_blocks)) return (int)cudaErrorInvalidValue;
  const int threads = rows <= 320 ? 320 : (rows + 31) / 32 * 32;      // (a thread looks up a CTA's first block, too)
  return (int)rx::launch(shared_plan_kernel, dim3(1), dim3(threads), 0, (cudaStream_t)stream, (const int*)row_seq, (const int*)ctx_len, (const int*)common, rows,
                         n_tables, max_blocks, n_q / n_kv, n_kv, (int*)plan, status);
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
  a.block_table = (const int*)block_table; a.plan = plan != nullptr ? (const int*)plan : own_plan;
  a.kv_scale = (const float*)kv_scale; a.status = status; a.max_blocks = max_blocks; a.n_q = n_q; a.n_kv = n_kv; a.rows = rows;
  a.n_tables = n_tables; a.scale_log2 = scale * 1.4426950408889634f;
  // Up to 64 rows are planned by every CTA of the attention for itself, which saves a launch (2.7 us of the host's 17.3 for a call) and the step from one kernel to the
  // next (64 rows behind 8192 common keys 45.1 -> 44.3 us, 57 drawn windows 18.3 -> 18.0 us); with more, the words that 296 CTAs write cost more (80 rows 26.0 against
  // 27.0 us, 182 rows 31 against 35 us).
  const bool here = plan == nullptr && rows <= SH_FUSED_ROWS;
  a.row_seq = here ? (const int*)row_seq : nullptr; a.ctx_len = (const int*)ctx_len; a.common = (const int*)common; a.planned = own_plan;
  if (plan == nullptr && !here) {
    const int r = rx_attn_shared_plan(row_seq, ctx_len, common, rows, n_tables, max_blocks, n_q, n_kv, own_plan, status, stream);
    if (r != 0) return r;
  }
  CUtensorMap tq;
  if (!sh_query_map(&tq, q, rows, n_q, n_q / n_kv, hd)) return (int)cudaErrorInvalidValue;
  const CUtensorMap &tk = *(const CUtensorMap*)tmap_k, &tv = *(const CUtensorMap*)tmap_v;
  if (hd == 128) e = kv_scale != nullptr ? launch_shared<128, true>(dev, tk, tv, tq, a, st) : launch_shared<128, false>(dev, tk, tv, tq, a, st);
  else e = kv_scale != nullptr ? launch_shared<64, true>(dev, tk, tv, tq, a, st) : launch_shared<64, false>(dev, tk, tv, tq, a, st);
  if (e != cudaSuccess) return (int)e;
  // (early whatever the grid: the kernel before is one wave of CTAs that do not wait for one another, and where one has ended the merge's next is there already)
  const long long blocks = n_q * hd / 128, merges = rows * blocks;
  const int split = merges <= SH_SPLIT16 && 4ll * max_blocks > SH_SPLIT16_OF ? 16 : merges <= SH_SPLIT4 ? 4 : 1;      // (each page may leave four)
  const auto merge = hd == 128 ? (split == 16 ? attn_shared_merge_kernel<128, 16, 16> : split == 4 ? attn_shared_merge_kernel<128, 4, 8> : attn_shared_merge_kernel<128, 1, 32>)
                               : (split == 16 ? attn_shared_merge_kernel<64, 16, 16> : split == 4 ? attn_shared_merge_kernel<64, 4, 8> : attn_shared_merge_kernel<64, 1, 16>);
  return (int)rx::launch_pdl(true, merge, dim3(rows, (unsigned)(split > 1 ? blocks : (blocks + 3) / 4)), dim3(split > 4 ? 32 * split : 128), 0, st, a.plan, a.part_o, a.part_ml, n_q, n_kv,
                             n_tables, max_blocks, (const __half*)suh, (__half*)xr, (uint16_t*)out);
}
