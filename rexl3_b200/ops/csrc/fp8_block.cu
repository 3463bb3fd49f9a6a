// Products of E4M3 rows with E4M3 weights, both under float32 scales for blocks of 128 (sm_100a).
//
//   out[r][n] = sum_b s[b][r] * ws[n / 128][b] * ( sum over the 128 k of block b of q[r][k] w[n][k] )   (+ bias[n])
//
// The inner sums are tensor-core products (kind::f8f6f4, float32 accumulators in tensor memory), one per block of k and from zero: a block's scales do not
// factor out of the sum over blocks.  So a group of warps takes each block's accumulator out of tensor memory, multiplies and adds it into registers
// while the next blocks' products fill the other accumulators.
#include <cuda.h>
#include "common.cuh"

namespace rx {

constexpr int FB_K = 128;                          // k of a block: one row of a 128-byte swizzled tile
constexpr int FB_A = 128 * FB_K;                   // bytes of a strip's block: 128 columns of the output
enum : int { FB_BF16 = 0, FB_F16 = 1, FB_F32 = 2 };

__device__ __forceinline__ void tc_mma_f8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
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
__device__ __forceinline__ void cp_async4(uint32_t dst, const float* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// one arrival once this thread's cp.async have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t pack2(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ float ld_cluster_f(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(mapa_u32(addr, rank)) : "memory");
  return v;
}

struct FbArgs {
  const float* s;            // [blocks of k][lds]
  const float* ws;           // [experts][strips][blocks of k]
  const float* bias;         // [N] or nullptr
  void* out;
  int* status;
  const int* offs;           // experts: [experts + 1] positions
  const int* src;            // position -> row * src_div (+ less than src_div), or nullptr: the row of its number
  const int* dst;            // position -> row of out, or nullptr
  long long lds, ldo;
  int rows, K, N, kblocks, out_type, experts, cap, src_div, out_rows;
};

template <typename V>
__device__ __forceinline__ void fb_store(const FbArgs& a, long long row, int n, V v) {
  const long long i = row * a.ldo + n;
  if (a.out_type == FB_BF16) ((__nv_bfloat16*)a.out)[i] = __float2bfloat16_rn(v);
  else if (a.out_type == FB_F16) ((__half*)a.out)[i] = __float2half_rn(v);
  else ((float*)a.out)[i] = v;
}

// Few rows.  The weights are the M side: a CTA has a strip of 128 output columns (TMEM lanes) and T rows (TMEM columns), and the CTAs of a cluster share the
// strip's blocks of k; their sums are added in the order of the CTAs through distributed shared memory.
template <int T>
struct FbStep {
  static constexpr int EW = T <= 64 ? 4 : 8;       // epilogue warps: four lane quarters, twice over 64 columns of 128 rows
  static constexpr int COLS = T * 4 / EW;          // accumulators of a thread
  static constexpr int THREADS = (EW + 3) * 32;
  static constexpr int STAGE = FB_A + T * FB_K;
  static constexpr int STAGES = T <= 32 ? 5 : T == 64 ? 4 : 6;
  static constexpr int BUFS = T == 128 ? 2 : 4;    // accumulators in tensor memory
  static constexpr int NCOLS = BUFS * T < 32 ? 32 : BUFS * T;
  static constexpr int SC = 8;                     // ring of scales: T of the rows, one of the strip
  static constexpr int SC_ROW = T + 4;
  static constexpr int SMEM = 1024 + STAGES * STAGE + SC * SC_ROW * 4 + 2 * T * 4 + 512;
};

template <int T, bool EXPERTS>
__global__ void __launch_bounds__(FbStep<T>::THREADS, T == 128 ? 1 : 2)
fp8_block_step_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ FbArgs a) {
  using L = FbStep<T>;
  pdl_launch();
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* scales = (float*)(smem + L::STAGES * L::STAGE);
  int* in_row = (int*)(scales + L::SC * L::SC_ROW);               // row of q that a row of the tile is, -1: none
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
    for (int i = 0; i < L::SC; ++i) { mbar_init(&sc_full[i], 32); mbar_init(&sc_empty[i], L::EW); }
    mbar_init(drained, 1);
    *abort_flag = 0;
    *n_sent = 0;
    fence_barrier_init();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_x);
  }
  for (int i = threadIdx.x; i < L::SC * L::SC_ROW; i += L::THREADS) scales[i] = 0.f;    // of rows that a tile lacks
  if (EXPERTS) {
    pdl_wait();                                    // the plan comes from a kernel before
    if (warp == 0) {
      // the expert whose rows hold the row_tile-th tile: experts' tiles counted up, 32 experts a step
      int before = 0, e = -1, pos = 0, n = 0;
      for (int e0 = 0; e0 < a.experts; e0 += 32) {
        const int i = e0 + lane;
        int lo = i < a.experts ? a.offs[i] : 0, hi = i < a.experts ? a.offs[i + 1] : 0;
        if (lo < 0 || hi < lo || hi > a.cap) {
          set_status(a.status, ST_BAD_ARG, 180, i);
          lo = hi = 0;
        }
        const int tiles = (hi - lo + T - 1) / T;
        int sum = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int u = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += u;
        }
        const int at = row_tile - before - (sum - tiles);         // which of the expert's tiles
        if (at >= 0 && at < tiles) e = i, pos = lo + at * T, n = min(T, hi - pos);
        before += __shfl_sync(0xffffffffu, sum, 31);
        if (before > row_tile) break;
      }
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

  uint64_t acc[L::COLS / 2];                                      // pairs of neighbouring rows
#pragma unroll
  for (int j = 0; j < L::COLS / 2; ++j) acc[j] = 0;
  const auto sum = [&acc](int j) { return __uint_as_float((uint32_t)(j & 1 ? acc[j >> 1] >> 32 : acc[j >> 1])); };

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
      for (int i = 0; i < nb; ++i) {
        const int s = i % L::STAGES;
        uint8_t* st = smem + s * L::STAGE;
        if (i >= L::STAGES) {
          if (!mbar_wait(&empty[s], ((i / L::STAGES) - 1) & 1, abort_flag, a.status, 183)) break;
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
      }
    }
  } else if (warp == L::EW + 1) {
    // ---- products
    if (!EXPERTS) pdl_wait();
    if (elect_one()) {
      constexpr uint32_t idesc = umma_idesc_e4m3(128, T);
      const uint64_t desc0 = umma_desc_k_sw128(smem_u32(smem));
      bool ok = true;
      for (int i = 0; i < nb && ok; ++i) {
        const int s = i % L::STAGES, buf = i % L::BUFS;
        if (i >= L::BUFS) ok = mbar_wait(&acc_empty[buf], ((i / L::BUFS) - 1) & 1, abort_flag, a.status, 184);
        if (ok) ok = mbar_wait(&full[s], (i / L::STAGES) & 1, abort_flag, a.status, 185);
        if (!ok) break;
        tc_fence_after();
        const uint64_t ad = desc0 + (uint64_t)((s * L::STAGE) >> 4), bd = ad + (FB_A >> 4);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f8(tmem + buf * T, ad + k * 2, bd + k * 2, idesc, k != 0);
        tc_commit(&empty[s]);
        tc_commit(&acc_full[buf]);
      }
      tc_commit(drained);                          // tensor memory is freed after the last product, also where another role gave up
      ring_landed(drained, 1, 1);
    }
  } else if (warp == L::EW + 2) {
    // ---- scales
    if (!EXPERTS) pdl_wait();
    const float* ws = a.ws + ((long long)expert * ((a.N + 127) / 128) + strip) * a.kblocks + b0;
    int mine[T >= 32 ? T / 32 : 1];
#pragma unroll
    for (int j = 0; j < T; j += 32) mine[j / 32] = j + lane < T ? in_row[j + lane] : -1;
    bool ok = true;
    for (int i = 0; i < nb && ok; ++i) {
      const int s = i % L::SC;
      if (i >= L::SC) ok = __all_sync(0xffffffffu, mbar_wait(&sc_empty[s], ((i / L::SC) - 1) & 1, abort_flag, a.status, 186, 20));
      if (!ok) break;
      const uint32_t slot = smem_u32(scales + s * L::SC_ROW);
#pragma unroll
      for (int j = 0; j < T; j += 32)
        if (mine[j / 32] >= 0) cp_async4(slot + (j + lane) * 4, a.s + (b0 + i) * a.lds + mine[j / 32]);
      if (lane == 0) cp_async4(slot + T * 4, ws + i);
      cp_async_arrive(&sc_full[s]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    // ---- sums: lane = column of the output
    if (!EXPERTS) pdl_wait();
    const int col0 = (warp >> 2) * L::COLS;
    const uint32_t src = tmem + ((uint32_t)((warp & 3) * 32) << 16) + col0;
    for (int i = 0; i < nb; ++i) {
      const int buf = i % L::BUFS, s = i % L::SC;
      bool ok = mbar_wait(&sc_full[s], (i / L::SC) & 1, abort_flag, a.status, 187);
      ok = ok && mbar_wait(&acc_full[buf], (i / L::BUFS) & 1, abort_flag, a.status, 188);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const float* sc = scales + s * L::SC_ROW;
      const float w = sc[T];
      const uint64_t w2 = pack2(w, w);
#pragma unroll
      for (int c = 0; c < L::COLS; c += 16) {
        uint32_t r[16];
        tc_ld_32x32b_x16(src + buf * T + c, r);
        tc_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sc + col0 + c + j);
          acc[(c + j) / 2] = fma2((uint64_t)r[j + 1] << 32 | r[j], mul2(pack2(f.x, f.y), w2), acc[(c + j) / 2]);
          acc[(c + j) / 2 + 1] = fma2((uint64_t)r[j + 3] << 32 | r[j + 2], mul2(pack2(f.z, f.w), w2), acc[(c + j) / 2 + 1]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&acc_empty[buf]);
        mbar_arrive(&sc_empty[s]);
      }
    }
    if (parts == 1 && *abort_flag == 0 && n < a.N) {
      const float bias = a.bias == nullptr ? 0.f : a.bias[n];
#pragma unroll
      for (int j = 0; j < L::COLS; ++j) {
        const int o = out_row[col0 + j];
        if (o >= 0) fb_store(a, o, n, (in_row[col0 + j] < 0 ? 0.f : sum(j)) + bias);
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
      for (int j = 0; j < L::COLS; ++j) red[((warp >> 2) * L::COLS + j) * 128 + (warp & 3) * 32 + lane] = sum(j);
    cluster_sync();
    const int j0 = T * part / parts, j1 = min(T * (part + 1) / parts, n_rows);
    const uint32_t base = smem_u32(red);
    for (int i = threadIdx.x; i < (j1 - j0) * 128; i += L::THREADS) {
      const int j = j0 + (i >> 7), c = strip * 128 + (i & 127);
      if (c >= a.N) continue;
      float v = 0.f;
      for (int r = 0; r < parts; ++r) v += ld_cluster_f(base + (j * 128 + (i & 127)) * 4, r);
      fb_store(a, row0 + j, c, v + (a.bias == nullptr ? 0.f : a.bias[c]));
    }
    cluster_sync();                                // nobody leaves while the others read
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

template <int T, bool EXPERTS>
static int fb_launch_step(const void* q, long long ldq, const void* w, const FbArgs& a, int row_tiles, int parts, cudaStream_t st) {
  using L = FbStep<T>;
  auto kern = fp8_block_step_kernel<T, EXPERTS>;
  CUtensorMap tw, tx;
  int e = fb_tmap(&tw, w, (uint64_t)a.N * (EXPERTS ? a.experts : 1), a.K, a.K, 128);
  if (e == 0) e = fb_tmap(&tx, q, a.rows, a.K, ldq, EXPERTS && a.src != nullptr ? 1 : T);
  if (e != 0) return e;
  static bool configured[64];                      // an attribute of the kernel on each device
  int dev = 0;
  cudaError_t ce = cudaGetDevice(&dev);
  if (ce == cudaSuccess && (dev >= 64 || !configured[dev])) {
    ce = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM);
    if (dev < 64) configured[dev] = ce == cudaSuccess;
  }
  if (ce != cudaSuccess) return (int)ce;
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

static int fb_check(const void* q, long long ldq, const FbArgs& a, const void* w) {
  if (a.rows < 1 || a.K < 16 || a.K % 16 != 0 || a.K > (1 << 24) || a.N < 1 || a.N > (1 << 22) || ldq < a.K || a.lds < a.rows || a.ldo < a.N) return (int)cudaErrorInvalidValue;
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
  a.s = (const float*)s, a.ws = (const float*)ws, a.bias = (const float*)bias, a.out = out, a.status = status;
  a.lds = lds, a.ldo = ldo, a.rows = rows, a.K = K, a.N = N, a.kblocks = (K + 127) / 128, a.out_type = out_type, a.experts = 1, a.out_rows = rows, a.src_div = 1;
  if (const int e = fb_check(q, ldq, a, w)) return e;
  cudaStream_t st = (cudaStream_t)stream;
  const int T = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 ? 64 : 128;
  const int row_tiles = (rows + T - 1) / T, strips = (N + 127) / 128;
  if (row_tiles > 65535 || strips > 65535) return (int)cudaErrorInvalidValue;
  const long long tiles = (long long)row_tiles * strips;
  int parts = (int)((T == 128 ? 148 : 296) / tiles);
  parts = parts > 8 ? 8 : parts;
  parts = parts > a.kblocks / 2 ? a.kblocks / 2 : parts;
  parts = parts < 1 ? 1 : parts;
  if (T == 16) return fb_launch_step<16, false>(q, ldq, w, a, row_tiles, parts, st);
  if (T == 32) return fb_launch_step<32, false>(q, ldq, w, a, row_tiles, parts, st);
  if (T == 64) return fb_launch_step<64, false>(q, ldq, w, a, row_tiles, parts, st);
  return fb_launch_step<128, false>(q, ldq, w, a, row_tiles, parts, st);
}

// w [experts][N][K], ws [experts][ceil(N / 128)][ceil(K / 128)]; offs int32 [experts + 1]: expert e has the positions offs[e] .. offs[e + 1] of `cap`.  Position p reads
// row src[p] / src_div of q (src nullptr: row p) and writes row dst[p] of out (dst nullptr: row p).
RX_API int rx_fp8_block_experts(const void* q, long long ldq, const void* s, long long lds, int rows, int K, const void* w, const void* ws, int experts, int N,
                                const void* offs, const void* src, int src_div, const void* dst, int cap, void* out, int out_type, long long ldo, int out_rows,
                                int* status, void* stream) {
  FbArgs a = {};
  a.s = (const float*)s, a.ws = (const float*)ws, a.out = out, a.status = status, a.offs = (const int*)offs, a.src = (const int*)src, a.dst = (const int*)dst;
  a.lds = lds, a.ldo = ldo, a.rows = rows, a.K = K, a.N = N, a.kblocks = (K + 127) / 128, a.out_type = out_type, a.experts = experts, a.cap = cap;
  a.src_div = src_div, a.out_rows = out_rows;
  if (const int e = fb_check(q, ldq, a, w)) return e;
  if (experts < 1 || experts > 4096 || (long long)experts * N > (1ll << 31) - 128 || cap < 1 || src_div < 1 || out_rows < 1 || offs == nullptr) return (int)cudaErrorInvalidValue;
  if ((src == nullptr && cap > rows) || (dst == nullptr && cap > out_rows)) return (int)cudaErrorInvalidValue;
  cudaStream_t st = (cudaStream_t)stream;
  const int each = (cap + experts - 1) / experts;  // rows of an expert on average
  const int T = each <= 16 ? 16 : each <= 32 ? 32 : each <= 64 ? 64 : 128;
  const int some = experts < cap ? experts : cap;
  const long long row_tiles = ((long long)cap + (long long)some * (T - 1)) / T;      // the most tiles that `cap` rows of `some` experts can make
  if (row_tiles > 65535) return (int)cudaErrorInvalidValue;
  if (T == 16) return fb_launch_step<16, true>(q, ldq, w, a, (int)row_tiles, 1, st);
  if (T == 32) return fb_launch_step<32, true>(q, ldq, w, a, (int)row_tiles, 1, st);
  if (T == 64) return fb_launch_step<64, true>(q, ldq, w, a, (int)row_tiles, 1, st);
  return fb_launch_step<128, true>(q, ldq, w, a, (int)row_tiles, 1, st);
}
