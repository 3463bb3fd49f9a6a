// Rows of E4M3 with a float32 scale for each block of 128 columns, for the products of fp8_block.cu (sm_100a).
//
//   add_norm     h += x (or + sum_t w_t x_t);  y = h * rsqrt(mean(h^2) + eps) * norm_w   (or y = h)
//   swiglu       y = silu(g) * u
//   both         s = max(max|y|, 2^-100) / 448 over a row's block,  q = e4m3(y / s):  q [rows][d] bytes, s [blocks][rows]
//
// All steps are float32; y is formed of the sum before that is rounded to h's type, and is rounded once, to its byte.  A thread holds eight neighbouring columns,
// so a block is 16 lanes: its largest magnitude is four shuffles, by maxima that keep a NaN, which so reaches the scale and the block.
// Scales stand block by block, rows side by side: the products read one block's scales of many rows at once, and a warp of them is one line.
#include <cuda_fp8.h>
#include "common.cuh"

namespace rx {

enum : int { F8R_BF16 = 0, F8R_F16 = 1, F8R_F32 = 2 };

// eight values from 16 (32) bytes at p + i; STREAM: they will not be read again
template <int T, bool STREAM = false>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&v)[8]) {
  if constexpr (T == F8R_F32) {
    const float4 a = *reinterpret_cast<const float4*>((const float*)p + i), b = *reinterpret_cast<const float4*>((const float*)p + i + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  } else {
    const uint4* from = reinterpret_cast<const uint4*>((const uint16_t*)p + i);
    const uint4 a = STREAM ? __ldcs(from) : *from;
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (T == F8R_BF16) {
        v[2 * j] = __uint_as_float(w[j] << 16), v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
        v[2 * j] = f.x, v[2 * j + 1] = f.y;
      }
    }
  }
}
__device__ __forceinline__ uint4 pack8_bf16(const float (&v)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    w[j] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
template <int T>
__device__ __forceinline__ void store8(void* p, size_t i, const float (&v)[8]) {
  if constexpr (T == F8R_F32) {
    *reinterpret_cast<float4*>((float*)p + i) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>((float*)p + i + 4) = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    *reinterpret_cast<uint4*>((uint16_t*)p + i) = pack8_bf16(v);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {         // NaN if either is
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
// g u / (1 + e^-g), a sixteenth of u over a sixteenth of the sum: from g = -87.3 down the reciprocal would be subnormal otherwise, which this form of it gives as 0.  (Instructions
// are what the kernel has least room for: the reciprocal that keeps them, 4097 x 14,336 55 -> 61 us; an exponential that does, 55 -> 57.)
__device__ __forceinline__ float silu_mul(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(fmaf(g, -1.4426950408889634f, -4.f)));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 0.0625f));
  return g * r * (0.0625f * u);
}
// The bytes of a thread's eight columns and, in `scale`, their block's scale.  The 16 lanes of a block call together (with zeros where the row has ended).
__device__ __forceinline__ uint2 to_e4m3(const float (&y)[8], float& scale) {
  float m = 7.888609052210118e-31f;                                // 2^-100: 1 / scale stays finite
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(y[j]));
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  constexpr float R = 1.f / 448.f;                                 // m / 448, corrected by its remainder (Markstein): as a division rounds
  scale = m * R;
  scale = fmaf(fmaf(-448.f, scale, m), R, scale);
  scale = m < __int_as_float(0x7F800000) ? scale : m;              // infinity, NaN: the remainder would be NaN
  float inv;                                                       // (within a step: of 448, the largest byte, what comes out above saturates)
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
  uint32_t w[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j] * inv, y[4 * j + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[4 * j + 2] * inv, y[4 * j + 3] * inv), __NV_SATFINITE, __NV_E4M3);
    w[j] = lo | hi << 16;
  }
  return make_uint2(w[0], w[1]);
}

struct NormArgs {
  const void* x;             // [rows][terms][d], rows ldx apart; nullptr: nothing is added
  const float* weights;      // [rows][terms], nullptr: one term of weight 1
  void* h;
  const uint16_t* norm_w;    // bf16 [d], nullptr: no norm
  uint8_t* q;
  float* s;
  uint16_t* xn;              // bf16 y, or nullptr
  long long ldx, ldh, ldq, lds, ldn;
  float eps, per_d;          // per_d: 1 / d
  int rows, terms, d;
};

// Bound by memory: every value is read and written once, and kept in registers in between.  8192 rows of 5120 (bf16) 52 us, 5.6 TB/s; 2100 rows of 2048 with 8 experts' outputs 14.6 us,
// 6.8 TB/s (part of it from L2); one row of 5120 2.0 us, all of it latency.
// NV vectors of eight columns a thread, kept in registers from the load to the bytes.  THREADS = 0: eight warps with a row each (narrow rows); otherwise one CTA a row.
enum : int { NORM_FIRST = 0, NORM_ADD = 1, NORM_EXPERTS = 2 };
template <int TX, int TH, int MODE, int NV, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS ? THREADS : 256, CTAS) add_norm_fp8_kernel(const __grid_constant__ NormArgs a) {
  pdl_launch();
  pdl_wait();
  __shared__ float sums[THREADS ? 32 : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = THREADS ? (int)threadIdx.x : lane, threads = THREADS ? (int)blockDim.x : 32;
  const long long row = THREADS ? (long long)blockIdx.x : (long long)blockIdx.x * 8 + warp;
  if (row >= a.rows) return;
  float y[NV][8];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * threads + t) * 8;
#pragma unroll
    for (int j = 0; j < 8; ++j) y[v][j] = 0.f;
    if (c < a.d) load8<TH>(a.h, row * a.ldh + c, y[v]);
  }
  if constexpr (MODE == NORM_ADD) {
    float x[NV][8];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * threads + t) * 8;
      if (c < a.d) load8<TX>(a.x, row * a.ldx + c, x[v]);
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * threads + t) * 8;
      if (c >= a.d) continue;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[v][j] += x[v][j];
      store8<TH>(a.h, row * a.ldh + c, y[v]);
    }
  } else if constexpr (MODE == NORM_EXPERTS) {
    constexpr int AT_ONCE = 4;                     // experts' outputs under way together
    for (int k0 = 0; k0 < a.terms; k0 += AT_ONCE) {
      float w[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) w[k] = k0 + k < a.terms ? a.weights[row * a.terms + k0 + k] : 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * threads + t) * 8;
        if (c >= a.d) continue;
        float x[AT_ONCE][8];
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k) {
#pragma unroll
          for (int j = 0; j < 8; ++j) x[k][j] = 0.f;
          if (w[k] != 0.f) load8<TX, true>(a.x, row * a.ldx + (long long)(k0 + k) * a.d + c, x[k]);
        }
#pragma unroll
        for (int k = 0; k < AT_ONCE; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) y[v][j] = fmaf(w[k], x[k][j], y[v][j]);
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * threads + t) * 8;
      if (c < a.d) store8<TH>(a.h, row * a.ldh + c, y[v]);
    }
  }
  float r = 1.f;
  if (a.norm_w != nullptr) {
    float sq = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < 8; ++j) sq = fmaf(y[v][j], y[v][j], sq);
    sq = warp_sum(sq);
    if constexpr (THREADS != 0) {
      if (lane == 0) sums[warp] = sq;
      __syncthreads();
      sq = warp_sum(lane < threads / 32 ? sums[lane] : 0.f);
    }
    r = rsqrtf(sq * a.per_d + a.eps);
  }
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c = (v * threads + t) * 8;
    if (a.norm_w != nullptr && c < a.d) {
      float w[8];
      load8<F8R_BF16>(a.norm_w, c, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[v][j] = y[v][j] * r * w[j];
    }
    float scale;
    const uint2 b = to_e4m3(y[v], scale);
    if (c < a.d) {
      *reinterpret_cast<uint2*>(a.q + row * a.ldq + c) = b;
      if ((t & 15) == 0) a.s[(long long)(c >> 7) * a.lds + row] = scale;
      if (a.xn != nullptr) *reinterpret_cast<uint4*>(a.xn + row * a.ldn + c) = pack8_bf16(y[v]);
    }
  }
}

struct SwigluArgs {
  const void* x;             // [rows][gate F | up F], rows ldx apart
  const int* total;          // rows that hold something, nullptr: all
  uint8_t* q;
  float* s;
  long long ldx, ldq, lds;
  int rows, F, blocks;       // blocks of a row
  uint32_t magic, shift;     // n / blocks = (umulhi(n, magic) + n) >> shift
};

// 16 lanes a block of 128 outputs, blocks row after row: a thread has eight outputs and no loop, so that a CTA's loads are all under way at once.  4097 rows of 14,336 (bf16) 48.5 us, 6.1 TB/s
// (a step over memory's time; the issue slots are nearly as full: an instruction more for each value costs 2 us); 64 rows of 17,408 2.5 us.
template <int TX>
__global__ void __launch_bounds__(256) swiglu_fp8_kernel(const __grid_constant__ SwigluArgs a) {
  pdl_launch();
  pdl_wait();
  const uint32_t n = blockIdx.x * 16 + (threadIdx.x >> 4), row32 = (__umulhi(n, a.magic) + n) >> a.shift;
  const long long row = row32;
  const int block = (int)(n - row32 * (uint32_t)a.blocks), c = block * 128 + (threadIdx.x & 15) * 8;
  const bool live = row < (a.total == nullptr ? a.rows : min(a.rows, *a.total)) && c < a.F;
  float y[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] = 0.f;
  if (live) {
    float g[8], u[8];
    load8<TX>(a.x, row * a.ldx + c, g);
    load8<TX>(a.x, row * a.ldx + a.F + c, u);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = silu_mul(g[j], u[j]);
  }
  float scale;
  const uint2 b = to_e4m3(y, scale);
  if (live) {
    *reinterpret_cast<uint2*>(a.q + row * a.ldq + c) = b;
    if ((threadIdx.x & 15) == 0) a.s[(long long)block * a.lds + row] = scale;
  }
}

template <int TX, int TH, int MODE, int NV, int THREADS, int CTAS>
static int launch_norm_as(const NormArgs& a, cudaStream_t st) {
  if (THREADS == 0) return (int)rx::launch(add_norm_fp8_kernel<TX, TH, MODE, NV, THREADS, CTAS>, dim3((a.rows + 7) / 8), dim3(256), 0, st, a);
  const int threads = ((a.d / 8 + NV - 1) / NV + 31) / 32 * 32;
  return (int)rx::launch(add_norm_fp8_kernel<TX, TH, MODE, NV, THREADS, CTAS>, dim3(a.rows), dim3(threads), 0, st, a);
}
// Narrow rows by a warp each, if there are enough of them: 20,000 rows of 512 10 us and not 21.5, but 64 2.06 and not 1.95; of 256 it is the faster one at any number.  Others by a CTA each, a thread a
// vector (1000 rows of 5120 6.9 us, with two a thread 8.0), and two or four past the 1024 threads that a CTA has.  With experts' outputs two, from 500 rows of more than 1024 on: half as many
// threads, each with eight loads under way and not four (1000 rows of 5120 19.9 and 25.2 us; 64 rows 4.4 and 3.3; 1000 of 1024 5.0 and 4.3).
template <int TX, int TH, int MODE>
static int launch_norm_mode(const NormArgs& a, cudaStream_t st) {
  if (a.d <= 256) return launch_norm_as<TX, TH, MODE, 1, 0, 1>(a, st);
  if constexpr (MODE != NORM_EXPERTS)
    if (a.d <= 512 && a.rows > 500) return launch_norm_as<TX, TH, MODE, 2, 0, 1>(a, st);
  if (a.d > 16384) return launch_norm_as<TX, TH, MODE, 4, 1024, 1>(a, st);
  if (a.d > 8192) return launch_norm_as<TX, TH, MODE, 2, 1024, 1>(a, st);
  if constexpr (MODE == NORM_EXPERTS)
    if (a.d > 1024 && a.rows > 500) return launch_norm_as<TX, TH, MODE, 2, 512, 2>(a, st);
  return launch_norm_as<TX, TH, MODE, 1, 1024, 1>(a, st);
}
template <int TX, int TH>
static int launch_norm(const NormArgs& a, cudaStream_t st) {
  if (a.x == nullptr) return launch_norm_mode<F8R_BF16, TH, NORM_FIRST>(a, st);
  if (a.weights == nullptr) return launch_norm_mode<TX, TH, NORM_ADD>(a, st);
  return launch_norm_mode<TX, TH, NORM_EXPERTS>(a, st);
}

}  // namespace rx

using namespace rx;

// x [rows][terms][d] (type x_type: 0 bf16, 1 fp16, 2 fp32) or nullptr, weights f32 [rows][terms] or nullptr (then terms = 1), h bf16 or fp32 (h_type 0 or 2),
// q bytes, s f32 [ceil(d / 128)][lds], xn bf16 or nullptr.  d a multiple of 16 up to 32768; every row begins on 16 bytes.
RX_API int rx_add_norm_fp8(const void* x, int x_type, long long ldx, const void* weights, int terms, void* h, int h_type, long long ldh, const void* norm_w, float eps,
                           void* q, long long ldq, void* s, long long lds, void* xn, long long ldn, int rows, int d, void* stream) {
  if (rows < 1 || rows > (1 << 30) || d < 16 || d % 16 != 0 || d > 32768 || terms < 1 || (terms > 1 && (weights == nullptr || x == nullptr))) return (int)cudaErrorInvalidValue;
  if (x_type < 0 || x_type > 2 || (h_type != F8R_BF16 && h_type != F8R_F32) || h == nullptr || q == nullptr || s == nullptr) return (int)cudaErrorInvalidValue;
  if (x != nullptr && ldx < (long long)terms * d || ldh < d || ldq < d || lds < rows || (xn != nullptr && ldn < d)) return (int)cudaErrorInvalidValue;
  if (((uintptr_t)x | (uintptr_t)h | (uintptr_t)q | (uintptr_t)xn | (uintptr_t)norm_w) & 15) return (int)cudaErrorMisalignedAddress;
  if (ldx * (x_type == F8R_F32 ? 4 : 2) % 16 || ldh * (h_type == F8R_F32 ? 4 : 2) % 16 || ldq % 16 || (xn != nullptr && ldn % 8)) return (int)cudaErrorMisalignedAddress;
  const NormArgs a = {x, (const float*)weights, h, (const uint16_t*)norm_w, (uint8_t*)q, (float*)s, (uint16_t*)xn, ldx, ldh, ldq, lds, ldn, eps, 1.f / (float)d, rows, terms, d};
  cudaStream_t st = (cudaStream_t)stream;
  if (h_type == F8R_BF16) {
    if (x_type == F8R_BF16) return launch_norm<F8R_BF16, F8R_BF16>(a, st);
    if (x_type == F8R_F16) return launch_norm<F8R_F16, F8R_BF16>(a, st);
    return launch_norm<F8R_F32, F8R_BF16>(a, st);
  }
  if (x_type == F8R_BF16) return launch_norm<F8R_BF16, F8R_F32>(a, st);
  if (x_type == F8R_F16) return launch_norm<F8R_F16, F8R_F32>(a, st);
  return launch_norm<F8R_F32, F8R_F32>(a, st);
}

// x [rows][2 F] (gate | up; type as above), q bytes [rows][F], s f32 [ceil(F / 128)][lds]; total: device int32, rows from it on are left as they are, or nullptr.
RX_API int rx_swiglu_fp8(const void* x, int x_type, long long ldx, void* q, long long ldq, void* s, long long lds, const void* total, int rows, int F, void* stream) {
  if (rows < 1 || F < 16 || F % 16 != 0 || F > (1 << 20) || x_type < 0 || x_type > 2 || x == nullptr || q == nullptr || s == nullptr) return (int)cudaErrorInvalidValue;
  if (ldx < 2ll * F || ldq < F || lds < rows) return (int)cudaErrorInvalidValue;
  if (((uintptr_t)x | (uintptr_t)q) & 15 || ldx * (x_type == F8R_F32 ? 4 : 2) % 16 || ldq % 16) return (int)cudaErrorMisalignedAddress;
  const int blocks = (F + 127) / 128;
  if ((long long)rows * blocks > 0x7FFFFFF0ll) return (int)cudaErrorInvalidValue;
  uint32_t shift = 0;
  while ((1u << shift) < (uint32_t)blocks) ++shift;
  const uint32_t magic = (uint32_t)((((1ull << shift) - blocks) << 32) / blocks + 1);
  const SwigluArgs a = {x, (const int*)total, (uint8_t*)q, (float*)s, ldx, ldq, lds, rows, F, blocks, magic, shift};
  const dim3 grid((uint32_t)(((long long)rows * blocks + 15) / 16)), threads(256);
  cudaStream_t st = (cudaStream_t)stream;
  if (x_type == F8R_BF16) return (int)rx::launch(swiglu_fp8_kernel<F8R_BF16>, grid, threads, 0, st, a);
  if (x_type == F8R_F16) return (int)rx::launch(swiglu_fp8_kernel<F8R_F16>, grid, threads, 0, st, a);
  return (int)rx::launch(swiglu_fp8_kernel<F8R_F32>, grid, threads, 0, st, a);
}
