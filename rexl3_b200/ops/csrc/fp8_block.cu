// Products of E4M3 rows with E4M3 weights, both under float32 scales for blocks of 128 (sm_100a).
//
//   out[r][n] = sum_b s[b][r] * ws[n / 128][b] * ( sum over the 128 k of block b of q[r][k] w[n][k] )   (+ bias[n])
//
// The inner sums are tensor-core products (kind::f8f6f4, float32 accumulators in tensor memory), one per block of k and from zero: a block's scales do not
// factor out of the sum over blocks.  So a group of warps takes each block's accumulator out of tensor memory, multiplies and adds it into registers
// while the next blocks' products fill the other accumulators.  Nothing is rounded to fewer than 32 bits before out.
//
// Two kernels.  Few rows: fp8_block_step_kernel, whose tensor-core rows are the weights' (128 columns of out) and whose columns are the rows (16, 32 or 64), so that a tile
// of few rows wastes nothing; it is bound by the weights' way from memory.  Many rows: fp8_block_wide_kernel, tiles of 128 x 256 or, by pairs of CTAs, 256 x 256.  Each has a form
// for routed experts.  An estimate of both chooses (below).
#include <cuda.h>
#include <math.h>
#include <type_traits>
#include "common.cuh"

namespace rx {

constexpr int FB_K = 128;                          // k of a block: one row of a 128-byte swizzled tile
constexpr int FB_A = 128 * FB_K;                   // bytes of a strip's block: 128 columns of the output
enum : int { FB_BF16 = 0, FB_F16 = 1, FB_F32 = 2 };

// the product of one block, 32 of its 128 k an instruction, from zero: a, b are the lower words of the operands' descriptors
template <int CG>
__device__ __forceinline__ void tc_mma_block(uint32_t d_tmem, uint32_t a, uint32_t b, uint32_t desc_hi, uint32_t idesc) {
#define RX_FB_MMA(G) asm volatile( \
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t" \
      "setp.ne.b32 p, 0, 0;\n\tsetp.eq.b32 q, 0, 0;\n\t" \
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t" \
      "tcgen05.mma.cta_group::" G ".kind::f8f6f4 [%0], a, b, %4, p;\n\t" \
      "add.u32 x, %1, 2;\n\tadd.u32 y, %2, 2;\n\tmov.b64 a, {x, %3};\n\tmov.b64 b, {y, %3};\n\t" \
      "tcgen05.mma.cta_group::" G ".kind::f8f6f4 [%0], a, b, %4, q;\n\t" \
      "add.u32 x, %1, 4;\n\tadd.u32 y, %2, 4;\n\tmov.b64 a, {x, %3};\n\tmov.b64 b, {y, %3};\n\t" \
      "tcgen05.mma.cta_group::" G ".kind::f8f6f4 [%0], a, b, %4, q;\n\t" \
      "add.u32 x, %1, 6;\n\tadd.u32 y, %2, 6;\n\tmov.b64 a, {x, %3};\n\tmov.b64 b, {y, %3};\n\t" \
      "tcgen05.mma.cta_group::" G ".kind::f8f6f4 [%0], a, b, %4, q;\n\t}" ::"r"(d_tmem), \
      "r"(a), "r"(b), "r"(desc_hi), "r"(idesc) \
      : "memory")
  if constexpr (CG == 2) RX_FB_MMA("2");
  else RX_FB_MMA("1");
#undef RX_FB_MMA
}
// both operands E4M3 (format 0) and K-major, float32 accumulators: the fields stand where umma_idesc_f16 has them
__host__ __device__ constexpr uint32_t umma_idesc_e4m3(int m, int n) { return umma_idesc_f16(m, n, 0, 0); }

// four rows of a tensor by their numbers, 128 bytes of each
__device__ __forceinline__ void tma_gather4(void* dst_smem, const void* tmap, int x, int r0, int r1, int r2, int r3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst_smem)),
      "l"(tmap), "r"(smem_u32(bar)), "r"(x), "r"(r0), "r"(r1), "r"(r2), "r"(r3)
      : "memory");
}
// A wait that ends with the barrier's phase or when the CTA's abort flag is up.  Few instructions, because a block's handing over waits four times: with a limit of its own in
// each (fb_watch has it for all) the loops ran out of the instruction cache, 270 cycles for a wait that was over before it began.
__device__ __forceinline__ bool fb_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .u32 f;\n\t"
      "POLL:\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "@p bra OVER;\n\t"
      "ld.volatile.shared.u32 f, [%3];\n\t"
      "setp.eq.u32 q, f, 0;\n\t"
      "@q bra POLL;\n\t"
      "OVER:\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity), "r"(smem_u32((const void*)abort_flag))
      : "memory");
  return ok != 0;
}
// One thread of the CTA, until `drained` (its last phase's end): puts the abort flag up when the host does, or when the copies have not come on for as long as a wait may last.
__device__ __forceinline__ void fb_watch(uint64_t* drained, const volatile int* progress, volatile int* abort_flag, int* status, int site) {
  const uint64_t limit = wait_limit_ns(status);
  uint64_t t0 = globaltimer_ns();
  int seen = *progress;
  for (uint32_t polls = 1; !mbar_try_wait(drained, 0); ++polls) {
    if (*abort_flag != 0) {
      ring_landed(drained, 1, 1);
      return;
    }
    if ((polls & 63u) != 0) continue;
    const uint64_t now = globaltimer_ns();
    if (*progress != seen) seen = *progress, t0 = now;
    const bool stop = host_abort(status);
    if (stop || now - t0 > limit) {
      set_status(status, stop ? ST_ABORTED : ST_TIMEOUT, site, seen);
      *abort_flag = 1;
    }
  }
}
// ... of a warp that works far ahead: one lane looks, now and then, and leaves the pipes to the others
__device__ __forceinline__ bool fb_wait_ahead(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  int ok = 1;
  if ((threadIdx.x & 31) == 0)
    while (!mbar_try_wait(bar, parity)) {
      if (*abort_flag != 0) {
        ok = 0;
        break;
      }
      __nanosleep(40);
    }
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}
// one arrival of a warp, by a predicate: a branch that parts its lanes costs 130 cycles
__device__ __forceinline__ void fb_arrive_warp(uint32_t bar) {
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar) : "memory");
}
// ... of all lanes of a warp
__device__ __forceinline__ bool fb_wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag) { return __all_sync(0xffffffffu, fb_wait(bar, parity, abort_flag)); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const uint8_t* src, int bytes) {      // 16 bytes, of which the last 16 - bytes are 0
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// one arrival once this thread's cp.async have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ float ld_cluster_f(uint32_t addr) {         // of an address that mapa gave
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void st_cluster_f4(uint32_t addr, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

// 16 or 32 columns of a thread's tensor memory lane
__device__ __forceinline__ void fb_ld(uint32_t taddr, uint32_t (&r)[16]) { tc_ld_32x32b_x16(taddr, r); }
__device__ __forceinline__ void fb_ld(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, "
      "%22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
        "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// the loads before have arrived; what uses r stays behind the wait
template <int N>
__device__ __forceinline__ void fb_ld_wait(uint32_t (&r)[N]) {
  tc_wait_ld();
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}

struct FbArgs {
  const uint8_t* q;          // [rows][K], rows ldq apart
  const float* s;            // [blocks of k][lds]
  const float* ws;           // [experts][strips][blocks of k]
  const float* bias;         // [N] or nullptr
  void* out;
  int* status;
  const int* offs;           // experts: [experts + 1] positions
  const int* src;            // position -> row * src_div (+ less than src_div), or nullptr: the row of its number
  const int* dst;            // position -> row of out, or nullptr
  long long ldq, lds, ldo;
  int rows, K, N, kblocks, out_type, experts, cap, src_div, out_rows;
};

template <typename V>
__device__ __forceinline__ void fb_store(const FbArgs& a, long long row, int n, V v) {
  const long long i = row * a.ldo + n;
  if (a.out_type == FB_BF16) ((__nv_bfloat16*)a.out)[i] = __float2bfloat16_rn(v);
  else if (a.out_type == FB_F16) ((__half*)a.out)[i] = __float2half_rn(v);
  else ((float*)a.out)[i] = v;
}

// A warp counts the experts' tiles of ROWS rows up, four experts a lane (their offsets arrive together): each(expert, tiles before its, its tiles, its positions) of those
// that there are; all tiles.  An expert whose offsets descend or leave the positions has none.
template <int ROWS, typename F>
__device__ __forceinline__ int fb_count_tiles(const FbArgs& a, int lane, F&& each) {
  int before = 0;
  for (int e0 = 0; e0 < a.experts; e0 += 128) {
    int o[5], tiles[4], mine = 0;
#pragma unroll
    for (int u = 0; u < 5; ++u) o[u] = a.offs[min(e0 + 4 * lane + u, a.experts)];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool good = o[u] >= 0 && o[u + 1] >= o[u] && o[u + 1] <= a.cap;
      if (!good && e0 + 4 * lane + u < a.experts) set_status(a.status, ST_BAD_ARG, 180, e0 + 4 * lane + u);
      tiles[u] = good ? (o[u + 1] - o[u] + ROWS - 1) / ROWS : 0;
      mine += tiles[u];
    }
    int sum = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, sum, d);
      if (lane >= d) sum += v;
    }
    int at = before + sum - mine;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (e0 + 4 * lane + u < a.experts) each(e0 + 4 * lane + u, at, tiles[u], o[u], o[u + 1]);
      at += tiles[u];
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  return before;
}

// Few rows.  The weights are the M side: a CTA has a strip of 128 output columns (TMEM lanes) and T rows (TMEM columns), and the CTAs of a cluster share the
// strip's blocks of k; their sums are added in the order of the CTAs through distributed shared memory.
// What bounds it: memory.  1 x 5120 -> 34,816 27.6 us, 6.5 TB/s (what a copy takes); 16 rows x 8 of 128 experts, 2048 -> 1536, 41 us, 6.3 TB/s.  A CTA's block takes 0.19 to 0.28 us of handing
// over (blocks by fours: one by one it was 0.5), so a strip with many blocks of k goes to several CTAs, which T = 64 has room for by whole clusters only: 64 x 17,408 -> 5120 has 40 strips
// in 3 parts, 120 of 148 SMs, 20.6 us, 4.4 TB/s.  Two CTAs of T = 64 an SM (four stages, batches of two): 30 us.
template <int T>
struct FbStep {
  static constexpr int PER_SM = T <= 32 ? 2 : 1;   // CTAs of an SM
  static constexpr int EW = T <= 32 ? 4 : 8;       // warps that take the sums: four lane quarters, for T > 32 of half the columns each
  static constexpr int COLS = 4 * T / EW;          // accumulators of a thread
  static constexpr int G = 4;                      // blocks that are handed over together
  static constexpr int BUFS = 2;                   // batches of accumulators in tensor memory
  static constexpr int SET = COLS == 32 ? 32 : 16; // columns of tensor memory that a thread loads at once
  static constexpr int THREADS = (EW + 4) * 32;    // and a warp each for the copies, the products, the scales, the watch over the waits
  static constexpr int STAGE = FB_A + T * FB_K;
  static constexpr int STAGES = T <= 32 ? 5 : 8;
  static constexpr int NCOLS = BUFS * G * T;
  static constexpr int SC_ROW = T;                 // scales of a block: the rows' times the strip's
  static constexpr int SC = 4;                     // batches of scales in shared memory, and two more in registers
  static constexpr int SC_BUF = G * SC_ROW;
  static constexpr int SMEM = 1024 + STAGES * STAGE + SC * SC_BUF * 4 + 2 * T * 4 + 512;
};

template <int T, bool EXPERTS>
__global__ void __launch_bounds__(FbStep<T>::THREADS, FbStep<T>::PER_SM)
fp8_block_step_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ FbArgs a) {
  using L = FbStep<T>;
  pdl_launch();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales = (float*)(smem + L::STAGES * L::STAGE);
  int* in_row = (int*)(scales + L::SC * L::SC_BUF);               // row of q that a row of the tile is, -1: none
  int* out_row = in_row + T;                                      // row of out, -1: none
  uint64_t* full = (uint64_t*)(out_row + T);
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;
  uint64_t* acc_empty = acc_full + L::BUFS;
  uint64_t* sc_full = acc_empty + L::BUFS;
  uint64_t* sc_empty = sc_full + L::SC;
  uint64_t* drained = sc_empty + L::SC;
  uint32_t* tmem_slot = (uint32_t*)(drained + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* n_sent = (volatile int*)(tmem_slot + 2);          // stages whose copies were issued
  int* tile = (int*)(tmem_slot + 3);                              // expert, first position, rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // dense: (part of k, row tile, strip); experts: (part of k, strip, tile)
  const int parts = EXPERTS ? 1 : gridDim.x, part = EXPERTS ? 0 : blockIdx.x;
  const int strip = EXPERTS ? blockIdx.x : blockIdx.z, row_tile = blockIdx.y;
  const int b0 = (int)((long long)a.kblocks * part / parts), nb = (int)((long long)a.kblocks * (part + 1) / parts) - b0;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < L::BUFS; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], L::EW); }
    for (int i = 0; i < L::SC; ++i) { mbar_init(&sc_full[i], 1); mbar_init(&sc_empty[i], L::EW); }
    mbar_init(drained, 1);
    *abort_flag = 0;
    *n_sent = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (EXPERTS) {
    pdl_wait();                                    // the plan comes from a kernel before
    if (warp == 0) {
      int e = -1, pos = 0, n = 0;                  // the expert whose rows hold the row_tile-th tile
      fb_count_tiles<T>(a, lane, [&](int i, int before, int tiles, int lo, int hi) {
        const int at = row_tile - before;
        if (at >= 0 && at < tiles) e = i, pos = lo + at * T, n = min(T, hi - pos);
      });
      const unsigned found = __ballot_sync(0xffffffffu, e >= 0);
      const int who = found ? __ffs(found) - 1 : 0;
      e = __shfl_sync(0xffffffffu, e, who), pos = __shfl_sync(0xffffffffu, pos, who), n = __shfl_sync(0xffffffffu, n, who);
      if (lane == 0) tile[0] = e, tile[1] = pos, tile[2] = found ? n : 0;
    }
    __syncthreads();
    if (tile[2] == 0) return;
  }
  const int expert = EXPERTS ? tile[0] : 0, row0 = EXPERTS ? tile[1] : row_tile * T;
  const int n_rows = EXPERTS ? tile[2] : min(T, a.rows - row0);
  for (int j = threadIdx.x; j < T; j += L::THREADS) {
    int r = -1, o = -1;
    if (j < n_rows) {
      r = row0 + j, o = row0 + j;
      if (EXPERTS) {
        if (a.src != nullptr) {
          const int v = a.src[r];
          r = v < 0 ? -1 : v / a.src_div;
        }
        if (r < 0 || r >= a.rows) {
          set_status(a.status, ST_BAD_ARG, 181, r);
          r = -1;
        }
        if (a.dst != nullptr) o = a.dst[o];
        if (o < 0 || o >= a.out_rows) {
          set_status(a.status, ST_BAD_ARG, 182, o);
          o = -1;
        }
      }
    }
    in_row[j] = r, out_row[j] = o;
  }
  if (warp == L::EW + 1) {
    tmem_alloc(tmem_slot, L::NCOLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int n = strip * 128 + (warp & 3) * 32 + lane;             // the output column of an epilogue thread

  float acc[L::COLS];
#pragma unroll
  for (int j = 0; j < L::COLS; ++j) acc[j] = 0.f;

  if (warp == L::EW) {
    // ---- copies
    if (elect_one()) {
      const int wrow = expert * a.N + strip * 128;
      const int ahead = min(nb, L::STAGES);
      for (int i = 0; i < ahead; ++i) {            // the weights are nobody's output
        mbar_arrive_expect_tx(&full[i], L::STAGE);
        tma_load_2d(smem + i * L::STAGE, &tmap_w, (b0 + i) * FB_K, wrow, &full[i]);
      }
      if (!EXPERTS) pdl_wait();
      int s = 0;
      uint32_t phase = 1;                          // of the stage's release before
      for (int i = 0; i < nb; ++i) {
        uint8_t* st = smem + s * L::STAGE;
        if (i >= L::STAGES) {
          if (!fb_wait(&empty[s], phase, abort_flag)) break;
          mbar_arrive_expect_tx(&full[s], L::STAGE);
          tma_load_2d(st, &tmap_w, (b0 + i) * FB_K, wrow, &full[s]);
        }
        if (EXPERTS && a.src != nullptr) {
          for (int j = 0; j < T; j += 4)
            tma_gather4(st + FB_A + j * FB_K, &tmap_x, (b0 + i) * FB_K, max(in_row[j], 0), max(in_row[j + 1], 0), max(in_row[j + 2], 0), max(in_row[j + 3], 0), &full[s]);
        } else {
          tma_load_2d(st + FB_A, &tmap_x, (b0 + i) * FB_K, row0, &full[s]);
        }
        *n_sent = i + 1;
        if (++s == L::STAGES) s = 0, phase ^= 1;
      }
    }
  } else if (warp == L::EW + 1) {
    // ---- products
    if (!EXPERTS) pdl_wait();
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_e4m3(128, T);
      const uint64_t desc0 = umma_desc_k_sw128(smem_u32(smem));
      int s = 0, g = 0, buf = 0;
      uint32_t phase = 0, acc_phase = 1;           // acc_phase: of the batch's release before; the first ones have none
      for (int i = 0; i < nb; ++i) {
        if (g == 0 && i >= L::BUFS * L::G && !fb_wait(&acc_empty[buf], acc_phase, abort_flag)) break;
        if (!fb_wait(&full[s], phase, abort_flag)) break;
        tc_fence_after();
        const uint32_t ad = (uint32_t)desc0 + s * (L::STAGE >> 4);
        tc_mma_block<1>(tmem + (buf * L::G + g) * T, ad, ad + (FB_A >> 4), (uint32_t)(desc0 >> 32), idesc);
        tc_commit(&empty[s]);
        if (++s == L::STAGES) s = 0, phase ^= 1;
        if (++g == L::G || i == nb - 1) {
          tc_commit(&acc_full[buf]);
          g = 0;
          if (++buf == L::BUFS) buf = 0, acc_phase ^= 1;
        }
      }
      tc_commit(drained);                          // tensor memory is freed after the last product, also where another role gave up
      ring_landed(drained, 1, 1);
    }
  } else if (warp == L::EW + 3) {
    if (!EXPERTS) pdl_wait();
    if (lane == 0) fb_watch(drained, n_sent, abort_flag, a.status, 183);
  } else if (warp == L::EW + 2) {
    // ---- scales
    if (!EXPERTS) pdl_wait();
    const float* ws = a.ws + ((long long)expert * ((a.N + 127) / 128) + strip) * a.kblocks + b0;
    constexpr int PER = T >= 32 ? T / 32 : 1;      // rows of a lane
    const float* from[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const int r = 32 * j + lane < T ? in_row[32 * j + lane] : -1;
      from[j] = r < 0 ? nullptr : a.s + b0 * a.lds + r;
    }
    const int batches = (nb + L::G - 1) / L::G;
    float v[2][L::G][PER], w[2][L::G];
    const auto load = [&](int i, float (&v)[L::G][PER], float (&w)[L::G]) {
#pragma unroll
      for (int g = 0; g < L::G; ++g) {
        const int b = i * L::G + g;
        w[g] = b < nb ? ws[b] : 0.f;
#pragma unroll
        for (int j = 0; j < PER; ++j) v[g][j] = b < nb && from[j] != nullptr ? from[j][b * a.lds] : 0.f;
      }
    };
    const auto put = [&](int i, float (&v)[L::G][PER], float (&w)[L::G]) {
      const int at = i % L::SC;
      float* slot = scales + at * L::SC_BUF;
      if (i >= L::SC && !fb_wait_ahead(&sc_empty[at], ((i / L::SC) - 1) & 1, abort_flag)) return false;
#pragma unroll
      for (int g = 0; g < L::G; ++g)
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (32 * j + lane < T) slot[g * L::SC_ROW + 32 * j + lane] = v[g][j] * w[g];
      __syncwarp();
      if (lane == 0) mbar_arrive(&sc_full[at]);
      return true;
    };
    load(0, v[0], w[0]);
    load(1, v[1], w[1]);
    for (int i = 0; i < batches; i += 2) {
      if (!put(i, v[0], w[0])) break;
      load(i + 2, v[0], w[0]);
      if (i + 1 >= batches || !put(i + 1, v[1], w[1])) break;
      load(i + 3, v[1], w[1]);
    }
  } else {
    // ---- sums: lane = column of the output
    if (!EXPERTS) pdl_wait();
    const int col0 = (warp >> 2) * L::COLS;
    const uint32_t src = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col0;
    const int batches = (nb + L::G - 1) / L::G;
    for (int i = 0; i < batches; ++i) {
      const int buf = i % L::BUFS, at = i % L::SC, blocks = min(L::G, nb - i * L::G);
      if (!__all_sync(0xffffffffu, fb_wait(&sc_full[at], (i / L::SC) & 1, abort_flag) & fb_wait(&acc_full[buf], (i / L::BUFS) & 1, abort_flag))) break;
      tc_fence_after();
      const float* sc = scales + at * L::SC_BUF + col0;
      uint32_t from = src + buf * L::G * T;
#pragma unroll 1
      for (int g = 0; g < blocks; ++g, from += T, sc += L::SC_ROW) {
#pragma unroll
        for (int c = 0; c < L::COLS; c += L::SET) {
          uint32_t r[L::SET];
          fb_ld(from + c, r);
          float4 f[L::SET / 4];
#pragma unroll
          for (int j = 0; j < L::SET; j += 4) f[j / 4] = *reinterpret_cast<const float4*>(sc + c + j);
          fb_ld_wait(r);
#pragma unroll
          for (int j = 0; j < L::SET; j += 4) {    // (pairs in one fma.f32x2: slower beside loads from tensor memory, 510 and 335 cycles for 128 columns of eight warps)
            acc[c + j] = fmaf(__uint_as_float(r[j]), f[j / 4].x, acc[c + j]), acc[c + j + 1] = fmaf(__uint_as_float(r[j + 1]), f[j / 4].y, acc[c + j + 1]);
            acc[c + j + 2] = fmaf(__uint_as_float(r[j + 2]), f[j / 4].z, acc[c + j + 2]), acc[c + j + 3] = fmaf(__uint_as_float(r[j + 3]), f[j / 4].w, acc[c + j + 3]);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      fb_arrive_warp(smem_u32(&acc_empty[buf]));
      fb_arrive_warp(smem_u32(&sc_empty[at]));
    }
    if (parts == 1 && *abort_flag == 0 && n < a.N) {
      const float bias = a.bias == nullptr ? 0.f : a.bias[n];
#pragma unroll
      for (int j = 0; j < L::COLS; ++j) {
        const int o = out_row[col0 + j];
        if (o >= 0) fb_store(a, o, n, (in_row[col0 + j] < 0 ? 0.f : acc[j]) + bias);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (*abort_flag != 0) {                          // copies may be under way, and must not outlive the CTA
    if (threadIdx.x == 0) ring_landed(full, L::STAGES, *n_sent);
    __syncthreads();
  }
  if (warp == L::EW + 1) {
    __syncwarp();
    tmem_dealloc(tmem, L::NCOLS);
  }
  if (parts > 1) {
    float* red = (float*)smem;                     // [T][128]: every copy of the ring has been read
    if (warp < L::EW)
#pragma unroll
      for (int j = 0; j < L::COLS; ++j) red[((warp >> 2) * L::COLS + j) * 128 + (warp & 3) * 32 + lane] = acc[j];
    cluster_sync();
    const int j0 = T * part / parts, j1 = min(T * (part + 1) / parts, n_rows);
    const uint32_t base = smem_u32(red);
    constexpr int AT_ONCE = 8;                     // sums of a thread whose loads are under way together: one after the other, each is a trip to another SM
    for (int i0 = threadIdx.x; i0 < (j1 - j0) * 128; i0 += L::THREADS * AT_ONCE) {
      float v[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) v[u] = 0.f;
      for (int r = 0; r < parts; ++r) {
        const uint32_t from = mapa_u32(base, r);
        float x[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          const int i = i0 + u * L::THREADS;
          x[u] = i < (j1 - j0) * 128 ? ld_cluster_f(from + (j0 * 128 + i) * 4) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) v[u] += x[u];
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const int i = i0 + u * L::THREADS, c = strip * 128 + (i & 127);
        if (i < (j1 - j0) * 128 && c < a.N) fb_store(a, row0 + j0 + (i >> 7), c, v[u] + (a.bias == nullptr ? 0.f : a.bias[c]));
      }
    }
    cluster_sync();                                // nobody leaves while the others read
  }
}

// Many rows.  The rows are the M side: a CTA has 128 rows (TMEM lanes) and 256 columns, alone (CG 1) or as half of a pair that shares the weights of a tile of
// 256 x 256 (CG 2).  A thread of the sums has one row, so a block's scale is one value for its 128 columns (a strip of the weights).  CTAs go from tile to tile; where
// there are few tiles, `parts` of them (pairs of them) in a cluster share a tile's blocks of k, and their sums are added in order through distributed shared memory.
// What bounds it: two accumulators of 256 columns are all of tensor memory, and one's round trip is the products (512 cycles), the sums (335: 128 multiply-adds and 8 loads of two warps
// a scheduler) and the barriers between (some 900): 890 cycles a block.  8192 x 5120 -> 34,816 1406 to 1510 us by the clock that the power leaves, 1.93 to 2.08 PFLOP/s; without the sums it would be
// 1125, without the products 960.  Slower: four accumulators of 128 columns (an operand is read from shared memory twice, 6%), 16 warps of sums (23%), one lane that waits for its warp (38%).
// Routed experts: 2100 rows x 8 of 128 experts, 2048 -> 1536, 145 us: what passes from L2 (800 MB, weights 1.5 times, because 131 rows an expert are two tiles for half of them).
template <int CG>
struct FbWide {
  static constexpr int EW = 8, THREADS = 384;      // 0-7: sums; 8: copies, 9: products, 10: scales, 11: the watch over the waits
  static constexpr int A = 128 * FB_K, B = 256 / CG * FB_K;
  static constexpr int STAGE = A + B, STAGES = CG == 2 ? 6 : 4;
  static constexpr int SG = 8, SC = 2;             // blocks of scales that are fetched and given back together; that many times
  static constexpr int SC_ROW = 132;               // of a block: 128 rows', two strips'
  static constexpr int SC_BUF = SG * SC_ROW + 260; // and, with a tile's first blocks, what the sums know of it: where each row goes, its row of q, the column tile
  static constexpr int MAX_EXPERTS = 4096;
  static constexpr int SMEM = 1024 + STAGES * STAGE + SC * SC_BUF * 4 + 512;
  static constexpr int SMEM_EXPERTS = SMEM + (MAX_EXPERTS + 1) * 4;
};

struct FbTile { int expert, row0, rows, ct; };     // rows of the tile (up to 128 CG), column tile

// expert whose rows make the row tile `rt`; first[e]: row tiles before expert e's
__device__ __forceinline__ int fb_expert_of(const int* first, int experts, int rt) {
  int lo = 0, hi = experts;                        // first[lo] <= rt < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (first[mid] <= rt) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <int CG>
__device__ __forceinline__ void fb_commit(uint64_t* bar, uint32_t rank) {
  if constexpr (CG == 2)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)(3u << (rank & ~1u))) : "memory");
  else
    tc_commit(bar);
}
// a copy into this CTA that reports to a barrier of the pair's first CTA
template <int CG>
__device__ __forceinline__ void fb_load(void* dst, const void* tmap, int x, int y, uint32_t bar) {
  if constexpr (CG == 2)
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(tmap), "r"(bar),
                 "r"(x), "r"(y)
                 : "memory");
  else
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(tmap), "r"(bar), "r"(x), "r"(y)
                 : "memory");
}
// Neighbouring columns of a row from n on.  A thread has a row, so value by value a warp would send 32 sectors for 64 bytes (200 x 4096 -> 2867: 24 us): WIDE, 32 bytes a store where every
// row begins on such a boundary; otherwise 16 bytes from the row's first 16-byte boundary on, shifted into place by selects, and what lies before it and behind the last one by itself.
template <int COLS>
__device__ __forceinline__ void fb_store_row(const FbArgs& a, long long row, int n, float (&acc)[COLS], bool zero, bool wide) {
  if (zero)
#pragma unroll
    for (int j = 0; j < COLS; ++j) acc[j] = 0.f;
  const int left = min(COLS, a.N - n);
  if (a.bias != nullptr) {
    const float* bias = a.bias + n;
#pragma unroll
    for (int j = 0; j < COLS; ++j)
      if (j < left) acc[j] += __ldg(bias + j);
  }
  const auto store = [&](auto type) {
    constexpr int TYPE = decltype(type)::value, SIZE = TYPE == FB_F32 ? 4 : 2, WORDS = COLS * SIZE / 4;
    const auto word = [&](int i) -> uint32_t {
      if (i >= WORDS) return 0u;
      if constexpr (TYPE == FB_F32) {
        return __float_as_uint(acc[i]);
      } else if constexpr (TYPE == FB_BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(acc[2 * i], acc[2 * i + 1]);
        return *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __floats2half2_rn(acc[2 * i], acc[2 * i + 1]);
        return *reinterpret_cast<const uint32_t*>(&h);
      }
    };
    char* p = (char*)a.out + (row * a.ldo + n) * SIZE;
    if ((SIZE == 2 || COLS < 128) && wide && left == COLS) {      // (of 128 float32 columns: the build would spill)
#pragma unroll
      for (int i = 0; i < WORDS; i += 8)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + 4 * i), "r"(word(i)), "r"(word(i + 1)), "r"(word(i + 2)), "r"(word(i + 3)), "r"(word(i + 4)),
                     "r"(word(i + 5)), "r"(word(i + 6)), "r"(word(i + 7))
                     : "memory");
      return;
    }
    const int before = (int)(-(uintptr_t)p & 15), end = left * SIZE - before;             // bytes; end: from the boundary on
    p += before;
    const auto some = [&](const uint32_t (&x)[4], int at, int from, int to) {      // of 16 bytes, the first of which is byte `at`, those from .. to
#pragma unroll
      for (int j = 0; j < 16 / SIZE; ++j) {
        const int b = at + SIZE * j;
        if (b < from || b >= to) continue;
        if constexpr (SIZE == 4) *reinterpret_cast<uint32_t*>(p + b) = x[j];
        else *reinterpret_cast<uint16_t*>(p + b) = (uint16_t)(j & 1 ? x[j / 2] >> 16 : x[j / 2]);
      }
    };
    if (before != 0) {
      const uint32_t x[4] = {word(0), word(1), word(2), word(3)};
      some(x, -before, -before, min(0, end));
    }
#pragma unroll
    for (int i = 0; i < WORDS; i += 4) {
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = word(i + j);
#pragma unroll
      for (int j = 0; j < 6; ++j) x[j] = before & 8 ? x[j + 2] : x[j];
#pragma unroll
      for (int j = 0; j < 5; ++j) x[j] = before & 4 ? x[j + 1] : x[j];
      if constexpr (SIZE == 2)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = __funnelshift_r(x[j], x[j + 1], before & 2 ? 16 : 0);
      const uint32_t y[4] = {x[0], x[1], x[2], x[3]};
      if (4 * i + 16 <= end) *reinterpret_cast<uint4*>(p + 4 * i) = make_uint4(y[0], y[1], y[2], y[3]);
      else if (4 * i < end) some(y, 4 * i, 4 * i, end);
    }
  };
  if (a.out_type == FB_BF16) store(std::integral_constant<int, FB_BF16>());
  else if (a.out_type == FB_F16) store(std::integral_constant<int, FB_F16>());
  else store(std::integral_constant<int, FB_F32>());
}

struct FbWideArgs { int parts, row_tiles, col_tiles, band, wide; };           // wide: every row of out begins on a 32-byte boundary

// Registers of a thread: what the block is launched with, and what the sums' warps and the others have then.  (Single CTAs that join their parts need a few more after the sums.)
constexpr int FB_WIDE_REGS = 168;
template <int CG, bool PARTS>
struct FbRegs {
  static constexpr int OTHERS = CG == 1 && PARTS ? 104 : 88, SUMS = CG == 1 && PARTS ? 200 : 208;
  static_assert(8 * SUMS + 4 * OTHERS <= 12 * FB_WIDE_REGS, "more registers than the block is launched with");
};

// PARTS: clusters of several parts, a tile each; otherwise a CTA (pair) goes from tile to tile.  (Both in one build: the sums' loop came out up to a quarter slower.)
template <int CG, bool EXPERTS, bool PARTS>
__global__ void __launch_bounds__(FbWide<CG>::THREADS, 1)
fp8_block_wide_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ FbArgs a, const __grid_constant__ FbWideArgs wa) {
  using L = FbWide<CG>;
  const int parts = PARTS ? wa.parts : 1;
  pdl_launch();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales = (float*)(smem + L::STAGES * L::STAGE);
  uint64_t* full = (uint64_t*)(scales + L::SC * L::SC_BUF);       // of the pair's first CTA: both CTAs' copies
  uint64_t* empty = full + L::STAGES;
  uint64_t* acc_full = empty + L::STAGES;
  uint64_t* acc_empty = acc_full + 2;                             // of the first CTA: both CTAs' sums
  uint64_t* sc_full = acc_empty + 2;
  uint64_t* sc_empty = sc_full + L::SC;
  uint64_t* drained = sc_empty + L::SC;
  uint32_t* tmem_slot = (uint32_t*)(drained + 1);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  volatile int* n_sent = (volatile int*)(tmem_slot + 2);          // stages that this CTA's copies were issued for
  int* sent = (int*)(tmem_slot + 3);                              // [STAGES] the bytes that the pair's second CTA copies for them
  int* first = (int*)(smem + L::SMEM - 1024);                     // experts: row tiles before each expert's
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank = 0;
  if (CG == 2 || PARTS) asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(rank));
  const int half = CG == 2 ? rank & 1 : 0, part = rank / CG, units = gridDim.x / (CG * parts), unit = blockIdx.x / (CG * parts);
  const int b0 = (int)((long long)a.kblocks * part / parts), nb = (int)((long long)a.kblocks * (part + 1) / parts) - b0;
  const uint32_t lead = CG == 2 ? rank & ~1u : rank;              // the pair's first CTA
  constexpr int ROWS = 128 * CG;

  if (threadIdx.x == 0) {
    for (int i = 0; i < L::STAGES; ++i) { mbar_init(&full[i], EXPERTS && a.src != nullptr ? 2 : 1); mbar_init(&empty[i], 1); }
    for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], CG * L::EW); }
    for (int i = 0; i < L::SC; ++i) { mbar_init(&sc_full[i], 32 + 1); mbar_init(&sc_empty[i], L::EW); }   // the scales' copies, the tile's rows
    mbar_init(drained, 1);
    *abort_flag = 0;
    *n_sent = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  if (warp == 9) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      tmem_alloc(tmem_slot, 512);
      tmem_relinquish();
    }
  }
  pdl_wait();
  if (EXPERTS && warp == 0) {
    const int all = fb_count_tiles<ROWS>(a, lane, [&](int i, int before, int, int, int) { first[i] = before; });
    if (lane == 0) first[a.experts] = all;
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2 || PARTS) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tiles = (EXPERTS ? first[a.experts] : wa.row_tiles) * wa.col_tiles;
  const auto tile_of = [&](int t) {
    FbTile f;
    if (EXPERTS) {
      const int rt = t / wa.col_tiles;
      f.ct = t - rt * wa.col_tiles;
      f.expert = fb_expert_of(first, a.experts, rt);
      const int lo = a.offs[f.expert], hi = a.offs[f.expert + 1];
      f.row0 = lo + (rt - first[f.expert]) * ROWS;
      f.rows = min(ROWS, hi - f.row0);
    } else {
      // through `band` row tiles, then to the next column tile
      const int b = t / (wa.band * wa.col_tiles), rb = min(wa.band, wa.row_tiles - b * wa.band), u = t - b * wa.band * wa.col_tiles;
      f.expert = 0;
      f.ct = u / rb;
      f.row0 = (b * wa.band + u % rb) * ROWS;
      f.rows = min(ROWS, a.rows - f.row0);
    }
    return f;
  };

  // waits until all but the last few of this warp's groups of copies have arrived, and shows the products the rows gathered for block number i
  constexpr int LATER = 1;
  const auto landed = [&](int i, auto later) {
    asm volatile("cp.async.wait_group %0;" ::"n"(decltype(later)::value) : "memory");
    fence_proxy_async();
    __syncwarp();
    if (lane == 0) mbar_arrive(&full[i % L::STAGES]);
  };
  // a group's registers are changed by all its four warps
  if (warp >= L::EW) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FbRegs<CG, PARTS>::OTHERS));
    if (warp == 8) {
      // ---- copies: this CTA's rows and its share of the tile's columns
      int s = 0, it = 0;
      uint32_t phase = 1;                          // of the stage's release before
      bool ok = true;
      for (int t = unit; t < tiles && ok; t += units) {
        const FbTile f = tile_of(t);
        const int mine = min(128, f.rows - 128 * half), others = CG == 2 ? min(128, f.rows - 128 * (half ^ 1)) : 0;
        const int row0 = f.row0 + 128 * half, wrow = f.expert * a.N + f.ct * 256 + (CG == 2 ? 128 * half : 0);
        if (EXPERTS && a.src != nullptr) {
          // Rows by their numbers, by ordinary 16-byte copies of the warp: eight lanes a row, a row's chunks where the copy engine's swizzle has them.  (The copy engine's own
          // gather of four rows takes 50 ns: 2100 rows x 8 picks of 128 experts, 2048 -> 1536, 206 -> 134 us.)
          // a division for each of four rows a lane; then row 4 j + lane / 8 comes from the lane that has it, in units of 16 bytes.  Rows that the tile lacks: its first.
          uint32_t own[4], off[32];
#pragma unroll
          for (int m = 0; m < 4; ++m) {
            const int at = 32 * m + lane, p = a.src[row0 + (at < mine ? at : 0)], d = p < 0 ? 0 : p / a.src_div;
            own[m] = d >= a.rows ? 0 : (uint32_t)(d * (a.ldq >> 4));                              // (the sums' threads report it)
          }
#pragma unroll
          for (int j = 0; j < 32; ++j) off[j] = __shfl_sync(0xffffffffu, own[j >> 3], (4 * j + (lane >> 3)) & 31);
          const uint32_t to = (lane >> 3) * FB_K, even = ((lane & 7) ^ (lane >> 3)) << 4, odd = ((lane & 7) ^ ((lane >> 3) + 4)) << 4;
          for (int b = 0; b < nb; ++b, ++it) {
            if (it >= L::STAGES && !fb_wait_ahead(&empty[s], phase, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* st = smem + s * L::STAGE;
            if (elect_one()) {
              *n_sent = it + 1;
              mbar_arrive_expect_tx(&full[s], L::B);
              fb_load<CG>(st + L::A, &tmap_w, (b0 + b) * FB_K, wrow, smem_u32(&full[s]));
            }
            __syncwarp();
            const int k = (b0 + b) * FB_K + (lane & 7) * 16, bytes = k < a.K ? 16 : 0;
            const uint8_t* from = a.q + (bytes ? k : 0);
            const uint32_t dst = smem_u32(st) + to;
#pragma unroll
            for (int m = 0; m < 4; ++m)
              if (32 * m < mine) {
#pragma unroll
                for (int j = 8 * m; j < 8 * m + 8; ++j) cp_async16(dst + j * 4 * FB_K + (j & 1 ? odd : even), from + off[j] * 16ull, bytes);
              }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (it >= LATER) landed(it - LATER, std::integral_constant<int, LATER>());
            if (++s == L::STAGES) s = 0, phase ^= 1;
          }
        } else {
          const uint32_t bytes = (mine > 0 ? L::A : 0) + L::B, both = bytes + (CG == 2 ? (others > 0 ? L::A : 0) + L::B : 0);
          for (int b = 0; b < nb; ++b, ++it) {
            if (it >= L::STAGES && !fb_wait_ahead(&empty[s], phase, abort_flag)) {
              ok = false;
              break;
            }
            uint8_t* st = smem + s * L::STAGE;
            const uint32_t bar = CG == 2 ? mapa_u32(smem_u32(&full[s]), lead) : smem_u32(&full[s]);
            if (elect_one()) {
              if (CG == 2) sent[s] = (int)(half == 0 ? both - bytes : bytes);
              *n_sent = it + 1;
              if (half == 0) mbar_arrive_expect_tx(&full[s], both);
              if (mine > 0) fb_load<CG>(st, &tmap_x, (b0 + b) * FB_K, row0, bar);
              fb_load<CG>(st + L::A, &tmap_w, (b0 + b) * FB_K, wrow, bar);
            }
            __syncwarp();
            if (++s == L::STAGES) s = 0, phase ^= 1;
          }
        }
      }
      if (EXPERTS && a.src != nullptr)             // the last stages' rows
        for (int i = max(0, it - LATER); i < it; ++i) landed(i, std::integral_constant<int, 0>());
    } else if (warp == 9) {
      // ---- products of the pair
      if (half == 0 && elect_one()) {
        int s = 0, buf = 0, it = 0;
        uint32_t phase = 0, acc_phase = 1;         // (of a barrier's phase before its first, a wait is over)
        constexpr uint32_t idesc = umma_idesc_e4m3(128 * CG, 256);
        const uint64_t desc0 = umma_desc_k_sw128(smem_u32(smem));
        bool ok = true;
        for (int t = unit; t < tiles && ok; t += units)
          for (int b = 0; b < nb; ++b, ++it) {
            ok = fb_wait(&full[s], phase, abort_flag) && fb_wait(&acc_empty[buf], acc_phase, abort_flag);
            if (!ok) break;
            tc_fence_after();
            const uint32_t ad = (uint32_t)desc0 + s * (L::STAGE >> 4);
            tc_mma_block<CG>(tmem + buf * 256, ad, ad + (L::A >> 4), (uint32_t)(desc0 >> 32), idesc);
            fb_commit<CG>(&acc_full[buf], rank);
            fb_commit<CG>(&empty[s], rank);
            if (++s == L::STAGES) s = 0, phase ^= 1;
            if (buf ^= 1; buf == 0) acc_phase ^= 1;
          }
        // nothing may still write the tensor memory that is freed, after a wait that gave up either
        fb_commit<CG>(drained, rank);
        ring_landed(drained, 1, 1);
      }
    } else if (warp == 11) {
      if (lane == 0) fb_watch(drained, n_sent, abort_flag, a.status, 190);
    } else if (warp == 10) {
      // ---- scales: four rows a lane, and the tile's two strips'.  (Rows that the tile lacks: whatever stands there, their sums go nowhere.)  And the tile's rows: the sums
      // would wait for their numbers with nothing else to do.
      int at = 0, it = 0;
      uint32_t phase = 1;
      bool ok = true;
      const int strips = (a.N + 127) / 128;
      for (int t = unit; t < tiles && ok; t += units) {
        const FbTile f = tile_of(t);
        const int mine = min(128, f.rows - 128 * half), row0 = f.row0 + 128 * half;
        const float* from[4];
        int in[4], out[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int n = 32 * j + lane;
          int r = n < mine ? row0 + n : -1, o = r;
          if (EXPERTS && r >= 0) {
            if (a.src != nullptr) {
              const int p = a.src[r];
              r = p < 0 ? -1 : p / a.src_div;
            }
            if (a.dst != nullptr) o = a.dst[o];
            if (r < 0 || r >= a.rows) {
              set_status(a.status, ST_BAD_ARG, 181, r);
              r = -1;
            }
            if (o < 0 || o >= a.out_rows) {
              set_status(a.status, ST_BAD_ARG, 182, o);
              o = -1;
            }
          }
          in[j] = r, out[j] = o;
          from[j] = r < 0 ? nullptr : a.s + (long long)b0 * a.lds + r;
        }
        const float* ws = a.ws + ((long long)f.expert * strips + 2 * f.ct + lane) * a.kblocks + b0;
        const bool strip = lane < 2 && 2 * f.ct + lane < strips;
        for (int b0g = 0; b0g < nb; b0g += L::SG, ++it) {
          if (it >= L::SC && !fb_wait_ahead(&sc_empty[at], phase, abort_flag)) {
            ok = false;
            break;
          }
          if (b0g == 0) {
            int* tile = (int*)(scales + at * L::SC_BUF + L::SG * L::SC_ROW);
#pragma unroll
            for (int j = 0; j < 4; ++j) tile[32 * j + lane] = out[j], tile[128 + 32 * j + lane] = in[j];
            if (lane == 0) tile[256] = f.ct;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sc_full[at]);
          const uint32_t slot = smem_u32(scales + at * L::SC_BUF + lane);
          for (int b = b0g; b < min(b0g + L::SG, nb); ++b) {
            const uint32_t to = slot + (b - b0g) * L::SC_ROW * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (from[j] != nullptr) cp_async4(to + 128 * j, from[j] + (long long)b * a.lds);
            if (strip) cp_async4(to + 512, ws + b);
          }
          cp_async_arrive(&sc_full[at]);
          if (++at == L::SC) at = 0, phase ^= 1;
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    __syncwarp();
    if (PARTS) cluster_sync();
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(FbRegs<CG, PARTS>::SUMS));
    // ---- sums: lane = row, warps 0-3 the tile's first 128 columns, 4-7 the others
    const int q = warp & 3, side = warp >> 2, at_row = 32 * q + lane;
    const uint32_t src = tmem + ((uint32_t)(q * 32) << 16) + 128 * side;
    const uint32_t acc_free = CG == 2 ? mapa_u32(smem_u32(acc_empty), lead) : smem_u32(acc_empty);
    int buf = 0, at = 0;
    uint32_t acc_phase = 0, sc_phase = 0;
    bool ok = true;
    for (int t = unit; t < tiles && ok; t += units) {
      ok = fb_wait_warp(&sc_full[at], sc_phase, abort_flag);
      if (!ok) break;
      const int* tile = (const int*)(scales + at * L::SC_BUF + L::SG * L::SC_ROW);
      const int o = tile[at_row], r = tile[128 + at_row], ct = tile[256];
      float acc[128];
#pragma unroll
      for (int j = 0; j < 128; ++j) acc[j] = 0.f;
      for (int b = 0; b < nb; ++b) {
        if (b % L::SG == 0 && b > 0) {
          ok = fb_wait_warp(&sc_full[at], sc_phase, abort_flag);
          if (!ok) break;
        }
        const float* sc = scales + at * L::SC_BUF + b % L::SG * L::SC_ROW;
        const float scale = sc[at_row] * sc[128 + side];
        ok = fb_wait_warp(&acc_full[buf], acc_phase, abort_flag);
        if (!ok) break;
        tc_fence_after();
        // the next 16 columns are on their way while these are added.  (All warps do all of it: a branch around it for rows that the tile lacks costs 8192 x 5120 -> 34,816 1553 and not
        // 1406 us, and without the loads ahead there are not registers enough.)
        uint32_t v[2][16];
        fb_ld(src + buf * 256, v[0]);
#pragma unroll
        for (int c = 0; c < 128; c += 16) {
          fb_ld_wait(v[c / 16 & 1]);
          if (c + 16 < 128) fb_ld(src + buf * 256 + c + 16, v[(c / 16 + 1) & 1]);
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[c + j] = fmaf(__uint_as_float(v[c / 16 & 1][j]), scale, acc[c + j]);
        }
        tc_fence_before();
        __syncwarp();
        fb_arrive_warp(acc_free + 8 * buf);
        if (buf ^= 1; buf == 0) acc_phase ^= 1;
        if ((b + 1) % L::SG == 0 || b == nb - 1) {
          fb_arrive_warp(smem_u32(&sc_empty[at]));
          if (++at == L::SC) at = 0, sc_phase ^= 1;
        }
      }
      if (!ok) break;
      const int n = ct * 256 + 128 * side;
      if (!PARTS) {
        if (o >= 0 && n < a.N) fb_store_row(a, o, n, acc, EXPERTS && r < 0, wa.wide != 0);
      } else {
        // One tile a cluster.  Once every CTA's ring has been read to its end, each part sends its sums of 16 columns to the part that adds them up (stores, which nobody waits for one by
        // one; fetched instead, 333 x 10,240 -> 1000 in 8 parts took 20.0 and not 17.5 us).  There they stand [part][16 columns][4 of them][128 rows][4].
        cluster_sync();
        const int most = (16 + parts - 1) / parts;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int group = 8 * side + i, owner = ((group + 1) * parts - 1) / 16;
          const uint32_t to = mapa_u32(smem_u32(smem), CG * owner + half) + (part * most + group - 16 * owner / parts) * (16 * 128 * 4) + at_row * 16;
#pragma unroll
          for (int u = 0; u < 4; ++u) st_cluster_f4(to + u * (128 * 16), acc[16 * i + 4 * u], acc[16 * i + 4 * u + 1], acc[16 * i + 4 * u + 2], acc[16 * i + 4 * u + 3]);
        }
      }
    }
    __syncwarp();
    if (PARTS && !ok) cluster_sync();
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2 && *abort_flag != 0 && threadIdx.x == 0)
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(smem_u32((const void*)abort_flag), rank ^ 1)), "r"(1) : "memory");
  __syncwarp();
  if (CG == 2 || PARTS) cluster_sync();
  if (*abort_flag != 0) {
    // Either CTA has given up, and the last copies may be under way.  A stage that only one CTA has issued its copies for gets the other's bytes here.
    if (half == 0 && threadIdx.x == 0) {
      const int n0 = *n_sent, n1 = CG == 2 ? ld_cluster((const int*)n_sent, lead + 1) : n0;
      for (int i = n1; i < n0; ++i)
        asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&full[i % L::STAGES])), "r"((uint32_t)sent[i % L::STAGES]) : "memory");
      for (int i = n0; i < n1; ++i) mbar_arrive_expect_tx(&full[i % L::STAGES], (uint32_t)ld_cluster(sent + i % L::STAGES, lead + 1));
      ring_landed(full, L::STAGES, max(n0, n1));
    }
    __syncwarp();
  } else if (PARTS) {
    // each of the parts adds up its share of the columns, a thread 16 neighbouring ones of a row at a time
    const FbTile f = tile_of(unit);
    const int row = threadIdx.x & 127, out_row = f.row0 + 128 * half + row, n0 = f.ct * 256;
    const int c1 = row < f.rows - 128 * half ? min(16 * (16 * (part + 1) / parts), a.N - n0) : 0;
    const int first_c = 16 * (16 * part / parts), most = (16 + parts - 1) / parts;
    for (int c = first_c + (threadIdx.x >> 7) * 16; c < c1; c += L::THREADS / 128 * 16) {
      const float4* from = (const float4*)smem + (c - first_c) / 16 * (4 * 128) + row;
      float v[16];
#pragma unroll
      for (int u = 0; u < 16; ++u) v[u] = 0.f;
      for (int p = 0; p < parts; ++p, from += most * (4 * 128))
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float4 x = from[u * 128];
          v[4 * u] += x.x, v[4 * u + 1] += x.y, v[4 * u + 2] += x.z, v[4 * u + 3] += x.w;
        }
      fb_store_row(a, out_row, n0 + c, v, false, wa.wide != 0);
    }
  }
  if (CG == 2) cluster_sync();
  if (warp == 9) {
    __syncwarp();
    if constexpr (CG == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    else tmem_dealloc(tmem, 512);
  }
}

typedef CUresult (*FbEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                               CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// byte rows `pitch` apart: boxes of 128 bytes x box_rows, swizzled; past the last row and the row's end stands 0
static int fb_tmap(CUtensorMap* out, const void* base, uint64_t rows, uint64_t cols, uint64_t pitch, uint32_t box_rows) {
  static FbEncodeFn enc = nullptr;
  if (enc == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return (int)cudaErrorNotSupported;
    enc = (FbEncodeFn)p;
  }
  cuuint64_t dims[2] = {cols, rows}, strides[1] = {pitch};
  cuuint32_t box[2] = {FB_K, box_rows}, estr[2] = {1, 1};
  const CUresult r = enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? 0 : (int)cudaErrorInvalidValue;
}

// lets a kernel have that much shared memory on the current device
template <auto KERN>
static int fb_allow(int smem) {
  static bool done[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !done[dev])) {
    e = cudaFuncSetAttribute(KERN, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (dev < 64) done[dev] = e == cudaSuccess;
  }
  return (int)e;
}

template <int T, bool EXPERTS>
static int fb_launch_step(const void* q, long long ldq, const void* w, const FbArgs& a, int row_tiles, int parts, cudaStream_t st) {
  using L = FbStep<T>;
  auto kern = fp8_block_step_kernel<T, EXPERTS>;
  CUtensorMap tw, tx;
  int e = fb_tmap(&tw, w, (uint64_t)a.N * (EXPERTS ? a.experts : 1), a.K, a.K, 128);
  if (e == 0) e = fb_tmap(&tx, q, a.rows, a.K, ldq, EXPERTS && a.src != nullptr ? 1 : T);
  if (e != 0) return e;
  if (const int ce = fb_allow<fp8_block_step_kernel<T, EXPERTS>>(L::SMEM)) return ce;
  const int strips = (a.N + 127) / 128;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = EXPERTS ? dim3(strips, row_tiles) : dim3(parts, row_tiles, strips);
  cfg.blockDim = dim3(L::THREADS), cfg.dynamicSmemBytes = L::SMEM, cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = EXPERTS ? 1 : parts, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() && (long long)parts * row_tiles * strips <= PDL_MAX_CTAS ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, tw, tx, a);
}

// The registers that the sums' warps add come out of what the block was launched with, and they would wait for them: a build with fewer a thread is not launched.
template <int CG, bool EXPERTS, bool PARTS>
static int fb_wide_builds() {
  static const int regs = [] {
    cudaFuncAttributes at;
    return cudaFuncGetAttributes(&at, fp8_block_wide_kernel<CG, EXPERTS, PARTS>) == cudaSuccess ? at.numRegs : 0;
  }();
  return regs == FB_WIDE_REGS ? 0 : (int)cudaErrorInvalidKernelImage;
}

template <int CG, bool EXPERTS, bool PARTS>
static int fb_launch_wide(const void* q, long long ldq, const void* w, const FbArgs& a, int parts, cudaStream_t st) {
  using L = FbWide<CG>;
  auto kern = fp8_block_wide_kernel<CG, EXPERTS, PARTS>;
  const int smem = EXPERTS ? L::SMEM_EXPERTS : L::SMEM;
  if (const int ce = fb_wide_builds<CG, EXPERTS, PARTS>()) return ce;
  if (const int ce = fb_allow<fp8_block_wide_kernel<CG, EXPERTS, PARTS>>(smem)) return ce;
  CUtensorMap tw, tx;
  int e = fb_tmap(&tw, w, (uint64_t)a.N * (EXPERTS ? a.experts : 1), a.K, a.K, 256 / CG);
  if (e == 0) e = fb_tmap(&tx, q, a.rows, a.K, ldq, 128);
  if (e != 0) return e;
  constexpr int ROWS = 128 * CG;
  FbWideArgs wa;
  wa.parts = parts;
  wa.col_tiles = (a.N + 255) / 256;
  const int some = a.experts < a.cap ? a.experts : a.cap;
  wa.row_tiles = EXPERTS ? (int)(((long long)a.cap + (long long)some * (ROWS - 1)) / ROWS) : (a.rows + ROWS - 1) / ROWS;
  const int bands = (wa.row_tiles + 8 / CG * 2 - 1) / (8 / CG * 2);
  wa.band = (wa.row_tiles + bands - 1) / bands;
  const int size = a.out_type == FB_F32 ? 4 : 2;
  wa.wide = ((uintptr_t)a.out | (uintptr_t)(a.ldo * size)) % 32 == 0;
  const long long tiles = (long long)wa.row_tiles * wa.col_tiles;
  if (tiles > (1 << 30)) return (int)cudaErrorInvalidValue;
  const int units = PARTS || tiles < 148 / CG ? (int)tiles : 148 / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CG * parts * units), cfg.blockDim = dim3(L::THREADS), cfg.dynamicSmemBytes = smem, cfg.stream = st;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CG * parts, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, tw, tx, a, wa);
}

// How many clusters of `size` CTAs of the kernel the current device holds at once with one CTA an SM.  (Clusters stay within a GPC: of six CTAs there is room for 22, of
// seven for 15.)
template <auto KERN>
static int fb_at_once(int dev, int size, int threads, int smem) {
  static int known[64][9];
  if (known[dev][size] == 0) {
    if (fb_allow<KERN>(smem) != 0) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(size), cfg.blockDim = dim3(threads), cfg.dynamicSmemBytes = smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = size, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    int n = 0;
    known[dev][size] = cudaOccupancyMaxActiveClusters(&n, KERN, &cfg) == cudaSuccess && n > 0 ? n : -1;
  }
  return known[dev][size];
}

// Which kernel a dense product takes, and how many parts of k: by an estimate of each one's microseconds, fitted to the times of all of them for 11 matrices (256 to 34,816 wide) at
// 18 row counts from 1 to 8192.  What it picks takes 0.9% longer than the fastest, on average (128 x 5120 -> 5120 the most: 18.2 us, 16.2).  A block of k takes a CTA of the few rows' kernel 0.19
// (T 16) to 0.28 us (T 64) and one of the other 0.41; memory gives 8 TB/s of weights and L2 22 of what tiles read again (parts of which other terms hide); a wave of the first starts in 4.4 us,
// the second in 4, and takes 1.8 a tile to begin and store; a cluster's sums cost 0.1 + 0.12 a part, and 2.2 + 0.9.
struct FbChoice { int cg, T, parts; double us; };
template <int T>
static void fb_consider_step(int dev, const FbArgs& a, FbChoice& best) {
  using L = FbStep<T>;
  const long long row_tiles = (a.rows + T - 1) / T, strips = (a.N + 127) / 128, tiles = row_tiles * strips;
  if (row_tiles > 65535) return;
  const double dram = (double)a.N * a.K, all = (double)tiles * a.kblocks * (FB_A + (a.rows < T ? a.rows : T) * FB_K), mem = dram / 8e6 + (all - dram) / 22e6;
  for (int parts = 1; parts <= 8 && parts <= a.kblocks; ++parts) {
    const int slots = L::PER_SM * fb_at_once<fp8_block_step_kernel<T, false>>(dev, parts, L::THREADS, L::SMEM);
    if (slots <= 0) continue;
    const double waves = (double)((tiles + slots - 1) / slots), blocks = (a.kblocks + parts - 1) / parts, k = waves * blocks * (T == 16 ? 0.19 : T == 32 ? 0.205 : 0.28);
    const double us = 4.4 * waves + sqrt(k * k + mem * mem) + (parts > 1 ? 0.1 + 0.12 * parts : 0);
    if (us < best.us) best = {0, T, parts, us};
  }
}
template <int CG>
static void fb_consider_wide(int dev, const FbArgs& a, FbChoice& best) {
  using L = FbWide<CG>;
  const long long row_tiles = (a.rows + 128 * CG - 1) / (128 * CG), tiles = row_tiles * ((a.N + 255) / 256);
  const double dram = (double)a.N * a.K, all = (double)tiles * CG * a.kblocks * ((a.rows < 128 ? a.rows : 128) * FB_K + L::B), mem = dram / 8e6 + (all - dram) / 22e6;
  for (int parts = 1; parts * CG <= 8 && parts <= a.kblocks; ++parts) {
    const int slots = parts > 1 ? fb_at_once<fp8_block_wide_kernel<CG, false, true>>(dev, CG * parts, L::THREADS, L::SMEM)
                                : fb_at_once<fp8_block_wide_kernel<CG, false, false>>(dev, CG, L::THREADS, L::SMEM);
    if (slots <= 0 || (parts > 1 && tiles > slots)) continue;      // (a cluster with parts has one tile)
    const double waves = (double)((tiles + slots - 1) / slots), blocks = (a.kblocks + parts - 1) / parts, k = waves * (blocks * 0.41 + 1.8);
    const double us = 4.0 + sqrt(k * k + mem * mem) + (parts > 1 ? 2.2 + 0.9 * parts : 0);
    if (us < best.us) best = {CG, 0, parts, us};
  }
}

static int fb_check(const void* q, long long ldq, const FbArgs& a, const void* w) {
  if (a.rows < 1 || a.rows > (1 << 30) || a.K < 16 || a.K % 16 != 0 || a.K > (1 << 24) || a.N < 1 || a.N > (1 << 22) || ldq < a.K || a.lds < a.rows || a.ldo < a.N) return (int)cudaErrorInvalidValue;
  if (q == nullptr || w == nullptr || a.s == nullptr || a.ws == nullptr || a.out == nullptr || a.out_type < 0 || a.out_type > 2) return (int)cudaErrorInvalidValue;
  if (((uintptr_t)q | (uintptr_t)w) & 15 || ldq % 16 || ((uintptr_t)a.s | (uintptr_t)a.ws | (uintptr_t)a.bias) & 3 ||
      (uintptr_t)a.out & (a.out_type == FB_F32 ? 3 : 1))
    return (int)cudaErrorMisalignedAddress;
  return 0;
}

}  // namespace rx

using namespace rx;

// q bytes [rows][K] (rows ldq apart), s f32 [ceil(K / 128)][lds], w bytes [N][K], ws f32 [ceil(N / 128)][ceil(K / 128)], bias f32 [N] or nullptr,
// out [rows][N] (rows ldo apart; type 0 bf16, 1 fp16, 2 fp32).
RX_API int rx_fp8_block_linear(const void* q, long long ldq, const void* s, long long lds, int rows, int K, const void* w, const void* ws, const void* bias, int N,
                               void* out, int out_type, long long ldo, int* status, void* stream) {
  FbArgs a = {};
  a.q = (const uint8_t*)q, a.ldq = ldq, a.s = (const float*)s, a.ws = (const float*)ws, a.bias = (const float*)bias, a.out = out, a.status = status;
  a.lds = lds, a.ldo = ldo, a.rows = rows, a.K = K, a.N = N, a.kblocks = (K + 127) / 128, a.out_type = out_type, a.experts = 1, a.out_rows = rows, a.src_div = 1;
  if (const int e = fb_check(q, ldq, a, w)) return e;
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return (int)e;
  if (dev >= 64) return (int)cudaErrorInvalidDevice;
  FbChoice c = {-1, 0, 0, 1e300};
  if (rows <= 16) fb_consider_step<16>(dev, a, c);
  else if (rows <= 32) fb_consider_step<32>(dev, a, c);
  else if (rows <= 512) fb_consider_step<64>(dev, a, c);
  if (rows > 16) {
    fb_consider_wide<1>(dev, a, c);
    fb_consider_wide<2>(dev, a, c);
  }
  cudaStream_t st = (cudaStream_t)stream;
  if (c.cg == 1) return c.parts > 1 ? fb_launch_wide<1, false, true>(q, ldq, w, a, c.parts, st) : fb_launch_wide<1, false, false>(q, ldq, w, a, 1, st);
  if (c.cg == 2) return c.parts > 1 ? fb_launch_wide<2, false, true>(q, ldq, w, a, c.parts, st) : fb_launch_wide<2, false, false>(q, ldq, w, a, 1, st);
  if (c.T == 16) return fb_launch_step<16, false>(q, ldq, w, a, 1, c.parts, st);
  if (c.T == 32) return fb_launch_step<32, false>(q, ldq, w, a, 1, c.parts, st);
  if (c.T == 64) return fb_launch_step<64, false>(q, ldq, w, a, (rows + 63) / 64, c.parts, st);
  return (int)cudaErrorInvalidConfiguration;
}

// w [experts][N][K], ws [experts][ceil(N / 128)][ceil(K / 128)]; offs int32 [experts + 1]: expert e has the positions offs[e] .. offs[e + 1] of `cap`.  Position p reads
// row src[p] / src_div of q (src nullptr: row p) and writes row dst[p] of out (dst nullptr: row p).
RX_API int rx_fp8_block_experts(const void* q, long long ldq, const void* s, long long lds, int rows, int K, const void* w, const void* ws, int experts, int N,
                                const void* offs, const void* src, int src_div, const void* dst, int cap, void* out, int out_type, long long ldo, int out_rows,
                                int* status, void* stream) {
  FbArgs a = {};
  a.q = (const uint8_t*)q, a.ldq = ldq, a.s = (const float*)s, a.ws = (const float*)ws, a.out = out, a.status = status, a.offs = (const int*)offs, a.src = (const int*)src, a.dst = (const int*)dst;
  a.lds = lds, a.ldo = ldo, a.rows = rows, a.K = K, a.N = N, a.kblocks = (K + 127) / 128, a.out_type = out_type, a.experts = experts, a.cap = cap;
  a.src_div = src_div, a.out_rows = out_rows;
  if (const int e = fb_check(q, ldq, a, w)) return e;
  if (experts < 1 || experts > FbWide<1>::MAX_EXPERTS || (long long)experts * N > (1ll << 31) - 128 || cap < 1 || cap > (1 << 30) || src_div < 1 || out_rows < 1 || offs == nullptr) return (int)cudaErrorInvalidValue;
  if ((src == nullptr && cap > rows) || (dst == nullptr && cap > out_rows)) return (int)cudaErrorInvalidValue;
  if (src != nullptr && (long long)rows * (ldq / 16) > 0xFFFFFFFFll) return (int)cudaErrorInvalidValue;      // a row's place is held in 32 bits, of 16 bytes
  cudaStream_t st = (cudaStream_t)stream;
  // Up to six positions an expert: tiles of 16 rows, whose CTAs begin sooner (8 of 128 experts, 2048 -> 1536: a row 10.2 us and 13.7, 768 positions 61 and 59, 2048 89 and 63; 2 of 16, 7168 -> 4096,
  // 24 rows 67 and 79).  But each of them begins anew, so with few blocks of k they have to find room at once (768 -> 2048: 24 positions 12.5 us and 13.4, 96 27.7 and 21).
  // And each of them counts all experts' tiles: 512 experts, 2048 -> 512, 128 positions 23.8 us and 26.7, 512 59.5 and 32; 4096 experts, 1536 -> 256, 4096 positions 768 and 62.
  const int some = experts < cap ? experts : cap;
  if (cap > 6 * experts || (long long)cap * experts > 65536 || (a.kblocks < 12 && (long long)some * ((N + 127) / 128) > 444)) return fb_launch_wide<1, true, false>(q, ldq, w, a, 1, st);
  const long long row_tiles = ((long long)cap + (long long)some * 15) / 16;          // the most tiles that `cap` rows of `some` experts can make
  return fb_launch_step<16, true>(q, ldq, w, a, (int)row_tiles, 1, st);
}
