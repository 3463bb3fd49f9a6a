// Sampling rules on logits, fused with the exact top candidates, and the token counts that they read (sm_100a).
//
// Counts: int16 [slots][vocab].  Bit 15 = the token stands in the prompt, bits 0 .. 14 = how often it was generated (it stops at 32767).
//
// Rules of a row, each step rounded to f32 in this order (no step is contracted with another, so that the order of near candidates is the definition's):
//     c    = generated count of the row's slot + how often the id is among the drafts that the window feeds before the row and at it
//     x    = seen ? (x > 0 ? x / repetition : x * repetition) : x            seen: in the prompt, or c > 0
//     x    = x - frequency * c;   x = x - (c > 0 ? presence : 0);   x = x + bias
//     x    = -inf where the row's grammar mask has no bit
// then the `count` best (value, then lower id).
#include "topk.cuh"

namespace rx {

// ------------------------------------------------------------------------------------------------ counts
constexpr int CNT_THREADS = 512;
constexpr int CNT_MAX_SLICE = 24576;                       // counters of a CTA: 96 KB of shared memory, two CTAs an SM
constexpr int CNT_MIN_SLICE = 1024;
constexpr unsigned CNT_PROMPT = 0x80000000u;

__device__ __forceinline__ uint16_t cnt_word(uint32_t c) {
  const uint32_t g = c & ~CNT_PROMPT;
  return (uint16_t)((g < 32767u ? g : 32767u) | (c >> 31 << 15));
}

// A CTA owns a slice of one slot's vocabulary: it reads the whole history, counts what falls into its slice in shared memory and writes the slice once.  No
// clearing pass, no atomics on global memory, one launch; what it costs is that a history is read once per slice, from L2 but for the first time.
__global__ void __launch_bounds__(CNT_THREADS) token_counts_kernel(uint16_t* __restrict__ counts, const int* __restrict__ slots, const int* __restrict__ starts,
                                                                   const int* __restrict__ prompt, const int* __restrict__ tokens, int n_tokens, int n_slots,
                                                                   int vocab, int slice, int* status) {
  pdl_launch();
  extern __shared__ uint32_t cnt[];
  const int req = blockIdx.y, tid = threadIdx.x;
  const int v0 = blockIdx.x * slice, v1 = min(vocab, v0 + slice);
  for (int i = tid; i < slice; i += CNT_THREADS) cnt[i] = 0;
  pdl_wait();
  const int slot = slots[req], begin = starts[req], end = starts[req + 1];
  bool skip = slot < 0 || slot >= n_slots || begin < 0 || end < begin || end > n_tokens;
  for (int j = tid; j < req; j += CNT_THREADS) skip |= slots[j] == slot;       // a slot twice: the first request's
  if (__syncthreads_or(skip)) {
    if (blockIdx.x == 0 && tid == 0) set_status(status, ST_BAD_ARG, 92, req);
    return;
  }
  const int p_end = begin + min(max(prompt[req], 0), end - begin);
  bool bad = false;
#pragma unroll 4
  for (int i = begin + tid; i < end; i += CNT_THREADS) {
    const int t = tokens[i];
    bad |= (unsigned)t >= (unsigned)vocab;
    if (t >= v0 && t < v1) {
      if (i < p_end) atomicOr(&cnt[t - v0], CNT_PROMPT);
      else atomicAdd(&cnt[t - v0], 1u);
    }
  }
  if (bad && blockIdx.x == 0) set_status(status, ST_BAD_ARG, 93, req);
  __syncthreads();
  // 16-byte stores where the slot's row allows them (rows of an odd vocabulary begin anywhere)
  uint16_t* out = counts + (size_t)slot * vocab;
  const int skew = (int)(((uintptr_t)(out + v0) >> 1) & 7), head = min(v1 - v0, (8 - skew) & 7), body = (v1 - v0 - head) & ~7;
  for (int i = tid; i < head; i += CNT_THREADS) out[v0 + i] = cnt_word(cnt[i]);
  for (int i = head + 8 * tid; i < head + body; i += 8 * CNT_THREADS) {
    uint32_t w[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) w[u] = (uint32_t)cnt_word(cnt[i + 2 * u]) | (uint32_t)cnt_word(cnt[i + 2 * u + 1]) << 16;
    *reinterpret_cast<uint4*>(out + v0 + i) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  for (int i = head + body + tid; i < v1 - v0; i += CNT_THREADS) out[v0 + i] = cnt_word(cnt[i]);
}

// counts[slots[i], tokens[i]] += 1 (or the prompt bit).  Compare-and-swap on the 16-bit word: the count stops at 32767, and the order does not matter.
__global__ void __launch_bounds__(256) token_counts_add_kernel(uint16_t* counts, const int* __restrict__ slots, const int* __restrict__ tokens, int n, int n_slots,
                                                               int vocab, int in_prompt, int* status) {
  pdl_launch();
  pdl_wait();
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const int slot = slots[i], t = tokens[i];
  if (slot < 0 || slot >= n_slots || t < 0 || t >= vocab) {
    set_status(status, ST_BAD_ARG, 94, i);
    return;
  }
  unsigned short* at = reinterpret_cast<unsigned short*>(counts) + (size_t)slot * vocab + t;
  unsigned short old = *reinterpret_cast<volatile unsigned short*>(at);
  while (true) {
    const unsigned short now = in_prompt ? (unsigned short)(old | 0x8000u) : (old & 0x7FFFu) == 0x7FFFu ? old : (unsigned short)(old + 1);
    if (now == old) return;
    const unsigned short was = atomicCAS(at, old, now);
    if (was == old) return;
    old = was;
  }
}

// ------------------------------------------------------------------------------------------------ rules + first selection
constexpr int PICK_MAX_BIAS = 1024;
struct PickArgs {
  const float* logits;                // row r at logits + r * ld
  const int* row_slot;                // [rows]; a value that is no slot: the row is under no penalties and no biases
  const uint16_t* counts;             // [n_slots][vocab] or nullptr
  const float* penalties;             // [n_slots][3]: repetition, frequency, presence
  const int* bias_id;                 // [n_slots][n_bias] or nullptr; a value that is no id: unused
  const float* bias_val;
  const uint32_t* mask;               // [n_masks][words] or nullptr; bit i of word w = id 32 w + i may be taken
  const int* mask_row;                // [rows]; a value that is no mask: every id may
  const int* first;                   // [rows] or nullptr: first row of the row's window
  const int* fed;                     // [rows]: token fed at the row
  uint64_t* cand;
  long long ld;
  int rows, vocab, n_slots, n_bias, n_masks, words, count, nchunks;
};

// A CTA takes 4096 ids of a row.  VEC: four ids side by side at a time (16-byte loads of logits, 8-byte loads of counts); else one.
// Masked ids cost neither their logit nor their count.  An id at -inf is no key at all (0): it is a candidate only where a row has fewer than `count` ids above
// -inf, and the second selection finds those by counting.  (As keys, thousands of equal values would all pass the selection's threshold.)
template <bool VEC>
__global__ void __launch_bounds__(TOPK_THREADS) pick_stage1_kernel(const __grid_constant__ PickArgs a) {
  pdl_launch();
  pdl_wait();
  __shared__ TopkShared sm;
  __shared__ float s_bias[TOPK_CHUNK];
  __shared__ uint16_t s_fed[TOPK_CHUNK];
  __shared__ uint32_t s_list[PICK_MAX_BIAS];              // biases inside this chunk: place in the slot's list << 12 | id - base, in no order
  __shared__ int s_listed;
  constexpr int W = VEC ? 4 : 1, N = TOPK_PER_THREAD / W;
  const int row = blockIdx.y, tid = threadIdx.x, base = blockIdx.x * TOPK_CHUNK;
  const int slot_in = a.row_slot != nullptr ? a.row_slot[row] : -1, slot = slot_in >= 0 && slot_in < a.n_slots ? slot_in : -1;
  const int mrow = a.mask != nullptr ? a.mask_row[row] : -1;
  const bool masked = mrow >= 0 && mrow < a.n_masks;
  // which of the thread's ids may be taken
  uint32_t ok = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int id = base + (i * TOPK_THREADS + tid) * W;
    if (id >= a.vocab) continue;
    const uint32_t w = masked ? a.mask[(size_t)mrow * a.words + (id >> 5)] >> (id & 31) : 0xFu;
    ok |= (w & ((1u << W) - 1)) << (i * W);
  }
  float x[TOPK_PER_THREAD];
  uint32_t c[TOPK_PER_THREAD];
  const float* lr = a.logits + (size_t)row * a.ld;
  const uint16_t* cr = a.counts != nullptr && slot >= 0 ? a.counts + (size_t)slot * a.vocab : nullptr;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int id = base + (i * TOPK_THREADS + tid) * W;
    const bool some = (ok >> (i * W) & ((1u << W) - 1)) != 0;
    if constexpr (VEC) {
      const float4 v = some ? *reinterpret_cast<const float4*>(lr + id) : make_float4(0.f, 0.f, 0.f, 0.f);
      const uint2 n = some && cr != nullptr ? *reinterpret_cast<const uint2*>(cr + id) : make_uint2(0u, 0u);
      x[4 * i] = v.x, x[4 * i + 1] = v.y, x[4 * i + 2] = v.z, x[4 * i + 3] = v.w;
      c[4 * i] = n.x & 0xFFFFu, c[4 * i + 1] = n.x >> 16, c[4 * i + 2] = n.y & 0xFFFFu, c[4 * i + 3] = n.y >> 16;
    } else {
      x[i] = some ? lr[id] : 0.f;
      c[i] = some && cr != nullptr ? cr[id] : 0u;
    }
  }
  // biases and drafts inside this chunk: rare, so the tables that hold them are only made where there are any
  const int* bid = a.bias_id != nullptr && slot >= 0 ? a.bias_id + (size_t)slot * a.n_bias : nullptr;
  const int nb = bid != nullptr ? a.n_bias : 0;
  const int r0 = a.first != nullptr && cr != nullptr ? max(a.first[row], 0) : row;
  if (tid == 0) s_listed = 0;
  __syncthreads();
  const int ids_here = min(a.vocab - base, TOPK_CHUNK);
  bool drafts = false;
  for (int e = tid; e < nb; e += TOPK_THREADS) {
    const int id = bid[e] - base;
    if (bid[e] >= 0 && id >= 0 && id < ids_here) s_list[atomicAdd(&s_listed, 1)] = (uint32_t)e << 12 | (uint32_t)id;
  }
  for (int r = r0 + 1 + tid; r <= row; r += TOPK_THREADS) drafts |= a.fed[r] >= base && a.fed[r] - base < ids_here;
  const bool any_drafts = __syncthreads_or(drafts);
  const int listed = s_listed;
  const bool any_bias = listed > 0;
  if (any_bias) for (int i = tid; i < TOPK_CHUNK; i += TOPK_THREADS) s_bias[i] = 0.f;
  if (any_drafts) for (int i = tid; i < TOPK_CHUNK / 2; i += TOPK_THREADS) reinterpret_cast<uint32_t*>(s_fed)[i] = 0u;
  __syncthreads();
  for (int i = tid; i < listed; i += TOPK_THREADS) {
    // an id that stands in the slot's list more than once: its first place adds them up in list order
    const uint32_t mine = s_list[i], id = mine & 4095u;
    float sum = a.bias_val[(size_t)slot * a.n_bias + (mine >> 12)];
    bool lead = true;
    for (uint32_t at = mine;;) {
      uint32_t next = ~0u;
      for (int j = 0; j < listed; ++j) {
        const uint32_t other = s_list[j];
        if ((other & 4095u) != id) continue;
        lead = lead && other >= mine;
        if (other > at && other < next) next = other;
      }
      if (!lead || next == ~0u) break;
      sum = __fadd_rn(sum, a.bias_val[(size_t)slot * a.n_bias + (next >> 12)]);
      at = next;
    }
    if (lead) s_bias[id] = sum;
  }
  if (drafts)
    for (int r = r0 + 1 + tid; r <= row; r += TOPK_THREADS) {
      const int id = a.fed[r] - base;
      if (a.fed[r] >= base && id < ids_here) atomicAdd(reinterpret_cast<uint32_t*>(s_fed) + (id >> 1), 1u << (16 * (id & 1)));
    }
  __syncthreads();
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (cr != nullptr) rep = a.penalties[3 * slot], freq = a.penalties[3 * slot + 1], pres = a.penalties[3 * slot + 2];
  uint64_t k[TOPK_PER_THREAD];
#pragma unroll
  for (int i = 0; i < TOPK_PER_THREAD; ++i) {
    const int local = ((i / W) * TOPK_THREADS + tid) * W + i % W;
    float v = x[i];
    const uint32_t gen = (c[i] & 0x7FFFu) + (any_drafts ? s_fed[local] : 0u);
    if (gen != 0 || c[i] != 0) {
      v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      v = __fsub_rn(v, __fmul_rn(freq, (float)gen));
      if (gen != 0) v = __fsub_rn(v, pres);
    }
    if (any_bias) v = __fadd_rn(v, s_bias[local]);
    v = v != v ? __uint_as_float(0x7FC00000u) : v + 0.f;  // every NaN is above +inf, and -0 is 0
    k[i] = (ok >> i & 1) && v != -INFINITY ? topk_key(v, (uint32_t)(base + local)) : 0;
  }
  block_select(k, a.count, a.cand + ((size_t)row * a.nchunks + blockIdx.x) * a.count, sm);
}

__global__ void __launch_bounds__(TOPK_THREADS) pick_stage2_kernel(const uint64_t* cand, int total, int count, int* __restrict__ ids, float* __restrict__ vals) {
  pdl_launch();
  pdl_wait();
  __shared__ TopkShared sm;
  __shared__ uint64_t outk[64];
  const int row = blockIdx.x;
  const uint64_t* c = cand + (size_t)row * total;
  uint64_t k[TOPK_PER_THREAD];
#pragma unroll
  for (int i = 0; i < TOPK_PER_THREAD; ++i) {
    const int j = i * TOPK_THREADS + threadIdx.x;
    k[i] = j < total ? c[j] : 0;
  }
  block_select(k, count, outk, sm);
  __syncthreads();
  if ((int)threadIdx.x >= count) return;
  int id;
  float v = -INFINITY;
  if (outk[threadIdx.x] != 0) {
    id = (int)(~(uint32_t)outk[threadIdx.x]);
    v = topk_val(outk[threadIdx.x]);
  } else {
    // fewer ids above -inf than places: the lowest of the other ids, which all stand at -inf, in order
    int n = 0;
    while (n < count && outk[n] != 0) ++n;
    int left = (int)threadIdx.x - n;                       // ids at -inf before this place's
    for (id = 0;; ++id) {
      bool taken = false;
      for (int j = 0; j < n; ++j) taken |= (int)(~(uint32_t)outk[j]) == id;
      if (!taken && left-- == 0) break;
    }
  }
  ids[(size_t)row * count + threadIdx.x] = id;
  vals[(size_t)row * count + threadIdx.x] = v;
}

}  // namespace rx

using namespace rx;

RX_API int rx_token_counts(void* counts, int n_slots, int vocab, const void* slots, const void* starts, const void* prompt, const void* tokens, int n_tokens, int n,
                           int* status, void* stream) {
  if (n < 1 || n > 65535 || n_slots < 1 || vocab < 1 || n_tokens < 0) return (int)cudaErrorInvalidValue;
  // slices so small that two waves of CTAs have work, so large that a history is not read more often than need be
  int slice = (vocab + (592 + n - 1) / n - 1) / ((592 + n - 1) / n);
  slice = slice < CNT_MIN_SLICE ? CNT_MIN_SLICE : slice > CNT_MAX_SLICE ? CNT_MAX_SLICE : (slice + 7) & ~7;
  const int parts = (vocab + slice - 1) / slice;
  static bool configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(token_counts_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CNT_MAX_SLICE * 4);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  return (int)rx::launch(token_counts_kernel, dim3(parts, n), dim3(CNT_THREADS), (size_t)slice * 4, (cudaStream_t)stream, (uint16_t*)counts, (const int*)slots,
                         (const int*)starts, (const int*)prompt, (const int*)tokens, n_tokens, n_slots, vocab, slice, status);
}

RX_API int rx_token_counts_add(void* counts, int n_slots, int vocab, const void* slots, const void* tokens, int n, int in_prompt, int* status, void* stream) {
  if (n < 1 || n_slots < 1 || vocab < 1) return (int)cudaErrorInvalidValue;
  return (int)rx::launch(token_counts_add_kernel, dim3((n + 255) / 256), dim3(256), 0, (cudaStream_t)stream, (uint16_t*)counts, (const int*)slots, (const int*)tokens, n,
                         n_slots, vocab, in_prompt, status);
}

// scratch: as rx_topk's.  Any of counts (with penalties), bias_id (with bias_val), mask (with mask_row) and first (with fed) may be null.
RX_API int rx_topk_adjusted(const void* logits, long long ld, int rows, int vocab, int count, void* scratch, void* ids, void* vals, const void* row_slot,
                            const void* counts, const void* penalties, int n_slots, const void* bias_id, const void* bias_val, int n_bias, const void* mask,
                            const void* mask_row, int n_masks, const void* first, const void* fed, void* stream) {
  const int nchunks = (vocab + TOPK_CHUNK - 1) / TOPK_CHUNK;
  if (rows < 1 || rows > 65535 || vocab < 1 || count < 1 || count > 64 || count > vocab || (long long)nchunks * count > TOPK_CHUNK || ld < vocab || n_bias < 0 || n_bias > PICK_MAX_BIAS)
    return (int)cudaErrorInvalidValue;
  PickArgs a = {(const float*)logits, (const int*)row_slot, (const uint16_t*)counts, (const float*)penalties, (const int*)bias_id, (const float*)bias_val,
                (const uint32_t*)mask, (const int*)mask_row, (const int*)first, (const int*)fed, (uint64_t*)scratch, ld, rows, vocab, n_slots, n_bias, n_masks,
                (vocab + 31) / 32, count, nchunks};
  // four ids at a time where every row of logits and counts begins on a 16- and an 8-byte boundary
  const bool vec = vocab % 4 == 0 && ld % 4 == 0 && ((uintptr_t)logits & 15) == 0 && ((uintptr_t)counts & 7) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  cudaError_t e = rx::launch(vec ? pick_stage1_kernel<true> : pick_stage1_kernel<false>, dim3(nchunks, rows), dim3(TOPK_THREADS), 0, st, a);
  if (e != cudaSuccess) return (int)e;
  return (int)rx::launch(pick_stage2_kernel, dim3(rows), dim3(TOPK_THREADS), 0, st, (const uint64_t*)scratch, nchunks * count, count, (int*)ids, (float*)vals);
}
