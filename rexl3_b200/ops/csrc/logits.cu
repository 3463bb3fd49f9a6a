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
#include "common.cuh"

namespace rx {

// ------------------------------------------------------------------------------------------------ counts
constexpr int CNT_THREADS = 1024;
constexpr int CNT_MAX_SLICE = 76032;                       // 16-bit words of a CTA: 152 KB of shared memory
constexpr int CNT_MIN_SLICE = 2048;
constexpr unsigned CNT_PROMPT = 0x80000000u;

// A CTA owns a slice of one slot's vocabulary: it reads the whole history, counts what falls into its slice in shared memory and writes the slice once.  No
// clearing pass, no atomics on global memory, one launch; what it costs is that a history is read once per slice, from L2 but for the first time.  The words are
// counted as they are stored, two in a 32-bit word of shared memory: with at most 32767 generated tokens no count can stop or carry.  A longer history takes
// the slice in two halves of 32-bit counters.
__global__ void __launch_bounds__(CNT_THREADS) token_counts_kernel(uint16_t* counts, const int* slots, const int* starts, const int* prompt,
                                                                   const int* tokens, int n_tokens, int n_slots, int vocab, int slice, int* status) {
  pdl_launch();
  extern __shared__ __align__(16) uint32_t cnt[];
  const int req = blockIdx.y, tid = threadIdx.x;
  const int v0 = blockIdx.x * slice, v1 = min(vocab, v0 + slice);
  auto clear = [&]() {
    for (int i = tid; i < slice / 8; i += CNT_THREADS) reinterpret_cast<uint4*>(cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
  };
  clear();
  pdl_wait();
  const int slot = slots[req], begin = starts[req], end = starts[req + 1];
  bool skip = slot < 0 || slot >= n_slots || begin < 0 || end < begin || end > n_tokens;
  for (int j = tid; j < req; j += CNT_THREADS) skip |= slots[j] == slot;       // a slot twice: the first request's
  if (__syncthreads_or(skip)) {
    if (blockIdx.x == 0 && tid == 0) set_status(status, ST_BAD_ARG, 92, req);
    return;
  }
  const int p_end = begin + min(max(prompt[req], 0), end - begin);
  uint16_t* out = counts + (size_t)slot * vocab;
  bool bad = false;
  if (end - p_end <= 32767) {
    // four tokens on their way at once
    for (int i0 = begin + tid; i0 < end; i0 += 4 * CNT_THREADS) {
      int t[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) t[u] = i0 + u * CNT_THREADS < end ? tokens[i0 + u * CNT_THREADS] : v0 - 1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (i0 + u * CNT_THREADS >= end) continue;
        bad |= (unsigned)t[u] >= (unsigned)vocab;
        if (t[u] < v0 || t[u] >= v1) continue;
        const int at = t[u] - v0;
        if (i0 + u * CNT_THREADS < p_end) atomicOr(&cnt[at >> 1], 0x8000u << (16 * (at & 1)));
        else atomicAdd(&cnt[at >> 1], 1u << (16 * (at & 1)));
      }
    }
    __syncthreads();
    // 16-byte stores where the slot's row allows them (rows of an odd vocabulary begin anywhere)
    const uint16_t* word = reinterpret_cast<const uint16_t*>(cnt);
    const int skew = (int)(((uintptr_t)(out + v0) >> 1) & 7), head = min(v1 - v0, (8 - skew) & 7), body = (v1 - v0 - head) & ~7;
    for (int i = tid; i < head; i += CNT_THREADS) out[v0 + i] = word[i];
    if (skew == 0) {
      for (int i = 8 * tid; i < body; i += 8 * CNT_THREADS) *reinterpret_cast<uint4*>(out + v0 + i) = *reinterpret_cast<const uint4*>(word + i);
    } else {
      for (int i = head + 8 * tid; i < head + body; i += 8 * CNT_THREADS) {
        uint32_t w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = (uint32_t)word[i + 2 * u] | (uint32_t)word[i + 2 * u + 1] << 16;
        *reinterpret_cast<uint4*>(out + v0 + i) = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    for (int i = head + body + tid; i < v1 - v0; i += CNT_THREADS) out[v0 + i] = word[i];
  } else {
    for (int h0 = v0; h0 < v1; h0 += slice / 2) {
      const int h1 = min(v1, h0 + slice / 2);
      for (int i = begin + tid; i < end; i += CNT_THREADS) {
        const int t = tokens[i];
        bad |= (unsigned)t >= (unsigned)vocab;
        if (t < h0 || t >= h1) continue;
        if (i < p_end) atomicOr(&cnt[t - h0], CNT_PROMPT);
        else atomicAdd(&cnt[t - h0], 1u);
      }
      __syncthreads();
      for (int i = tid; i < h1 - h0; i += CNT_THREADS) {
        const uint32_t g = cnt[i] & ~CNT_PROMPT;
        out[h0 + i] = (uint16_t)((g < 32767u ? g : 32767u) | (cnt[i] >> 31 << 15));
      }
      __syncthreads();
      clear();
      __syncthreads();
    }
  }
  if (bad && blockIdx.x == 0) set_status(status, ST_BAD_ARG, 93, req);
}

// counts[slots[i], tokens[i]] += 1 (or the prompt bit).  Compare-and-swap on the 16-bit word: the count stops at 32767, and the order does not matter.
__global__ void __launch_bounds__(256) token_counts_add_kernel(uint16_t* counts, const int* slots, const int* tokens, int n, int n_slots, int vocab,
                                                               int in_prompt, int* status) {
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
constexpr int PICK_MAX_BIAS = 1024, PICK_MAX_WINDOW = 4096;      // (a row looks through its slot's biases and its window's rows before it)
struct PickArgs {
  const float* logits;                // row r at logits + r * ld
  const int* row_slot;                // [rows]; a value that is no slot: the row is under no penalties and no biases
  const uint16_t* counts;             // [n_slots][vocab] or nullptr
  const float* penalties;             // [n_slots][3]: repetition, frequency, presence
  const int* bias_id;                 // [n_slots][n_bias] or nullptr; a value that is no id: unused
  const float* bias_val;
  const uint32_t* mask;               // [n_masks][words] or nullptr; bit i of word w = id 32 w + i may be taken
  const int* mask_row;                // [rows]; a value that is no mask: every id may
  const int* first;                   // [rows] or nullptr: first row of the row's window (below 0: 0; behind the row: the row)
  const int* fed;                     // [rows]: token fed at the row
  uint64_t* cand;
  int* ids;                           // of a vocabulary of one chunk of 4096: the results, without a second kernel; else nullptr
  float* vals;
  long long ld;
  int rows, vocab, n_slots, n_bias, n_masks, words, count, nchunks;
};

// The order of values as that of unsigned words (0: no candidate): every NaN is above +inf, -0 is 0.
__device__ __forceinline__ uint32_t pick_order(float v) {
  const uint32_t b = __float_as_uint(v != v ? __uint_as_float(0x7FC00000u) : v + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t pick_key(uint32_t order, int id) { return (uint64_t)order << 32 | (uint32_t)~id; }

// The rules but for the mask.
__device__ __forceinline__ float pick_rules(float v, uint32_t word, uint32_t drafts, float rep, float freq, float pres) {
  const uint32_t gen = (word & 0x7FFFu) + drafts;
  if (gen != 0 || word != 0) {
    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    v = __fsub_rn(v, __fmul_rn(freq, (float)gen));
    if (gen != 0) v = __fsub_rn(v, pres);
  }
  return v;
}

constexpr int PICK_THREADS = 256, PICK_CTAS = 5, PICK_LIST = 512;
struct PickShared { uint32_t best[PICK_THREADS], least; int n; uint64_t list[PICK_LIST], top[PICK_THREADS / 32]; };

// The `count` (<= 64) largest keys of the block, in descending order, to out, `apart` from one another (0 where there are fewer).  `mine` is the order of the thread's best (0: it has
// none); each(least, f) calls f(key) for the thread's keys whose order is at least `least` (> 0).
// As many threads as `count` have an order from the count-th largest of the threads' own best on, so no key with a lower order can be among the results.  One warp
// searches for that threshold by quartering the interval between the lowest and the highest best, and takes a lower one that few more threads pass: the steps that
// are left would cost more than the few keys.  Each key that passes finds its place by counting the larger ones.
// Where more pass than the list holds (many equal values, or one thread that has most of the high ones), the block's maximum is taken `count` times.
template <typename Each>
__device__ __forceinline__ void pick_select(uint32_t mine, Each each, int count, uint64_t* out, int apart, PickShared& sm) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  sm.best[tid] = mine;
  if (tid == 0) sm.n = 0;
  __syncthreads();
  if (warp == 0) {
    constexpr int K = PICK_THREADS / 32;
    uint32_t b[K], lo = ~0u, hi = 0;
    int pass = 0;                                          // threads from lo on; from hi + 1 on too few
#pragma unroll
    for (int i = 0; i < K; ++i) b[i] = sm.best[i * 32 + lane], lo = min(lo, b[i] - 1), hi = max(hi, b[i]), pass += b[i] != 0;
    lo = __reduce_min_sync(0xffffffffu, lo) + 1;           // (of those that have any)
    hi = __reduce_max_sync(0xffffffffu, hi);
    pass = __reduce_add_sync(0xffffffffu, pass);
    if (pass < count) lo = hi = 1;                         // all
    while (pass > count + count / 4 + 2 && lo < hi) {
      // three probes at once: a step's time is that of its chain
      const uint32_t q = (hi - lo) / 4, m1 = lo + q + 1, m3 = hi - q, m2 = m1 + (m3 - m1) / 2;
      int c1 = 0, c2 = 0, c3 = 0;
#pragma unroll
      for (int i = 0; i < K; ++i) c1 += b[i] >= m1, c2 += b[i] >= m2, c3 += b[i] >= m3;
      c1 = __reduce_add_sync(0xffffffffu, c1);
      c2 = __reduce_add_sync(0xffffffffu, c2);
      c3 = __reduce_add_sync(0xffffffffu, c3);
      if (c3 >= count) lo = m3, pass = c3;
      else if (c2 >= count) lo = m2, pass = c2, hi = m3 - 1;
      else if (c1 >= count) lo = m1, pass = c1, hi = m2 - 1;
      else hi = m1 - 1;
    }
    if (lane == 0) sm.least = lo;
  }
  __syncthreads();
  const uint32_t least = sm.least;
  if (mine >= least)
    each(least, [&](uint64_t key) {
      const int at = atomicAdd(&sm.n, 1);
      if (at < PICK_LIST) sm.list[at] = key;
    });
  __syncthreads();
  const int n = sm.n;
  if (n <= PICK_LIST) {
    for (int i = tid; i < n; i += PICK_THREADS) {
      const uint64_t own = sm.list[i];
      int place = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) place += sm.list[j] > own;
      if (place < count) out[place * apart] = own;
    }
    for (int r = n + tid; r < count; r += PICK_THREADS) out[r * apart] = 0;
    return;
  }
  uint64_t below = ~0ull, own = 0;                         // the last maximum; the thread's best that is below it
  bool again = mine != 0;
  for (int r = 0; r < count; ++r) {
    if (again) {
      own = 0;
      each(1u, [&](uint64_t key) { if (key < below) own = max(own, key); });
    }
    uint64_t best = own;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) sm.top[warp] = best;
    __syncthreads();
    below = 0;
#pragma unroll
    for (int w = 0; w < PICK_THREADS / 32; ++w) below = max(below, sm.top[w]);
    again = below != 0 && own == below;
    if (tid == 0) out[r * apart] = below;
    __syncthreads();
  }
}

// the value that a word stands for (not 0)
__device__ __forceinline__ float pick_value(uint32_t order) { return __uint_as_float(order & 0x80000000u ? order & 0x7FFFFFFFu : ~order); }
// the larger value; a NaN is above all
__device__ __forceinline__ float pick_max(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// A row's results, from its best keys (in order, 0 behind the last); taken[4] is 0
__device__ __forceinline__ void pick_finish(const uint64_t* outk, uint32_t* taken, int row, int count, int* ids, float* vals) {
  if ((int)threadIdx.x < count && outk[threadIdx.x] != 0) {
    const uint32_t own = ~(uint32_t)outk[threadIdx.x];
    if (own < 128) atomicOr(&taken[own >> 5], 1u << (own & 31));
  }
  __syncthreads();
  if ((int)threadIdx.x >= count) return;
  int id;
  float v = -INFINITY;
  if (outk[threadIdx.x] != 0) {
    id = (int)(~(uint32_t)outk[threadIdx.x]);
    v = pick_value((uint32_t)(outk[threadIdx.x] >> 32));
  } else {
    // Fewer ids above -inf than places: the lowest of the other ids, which all stand at -inf, in order.  With at most 64 ids to leave out they are below 128.
    int q = threadIdx.x, w = 0;
    for (int r = 0; r < count; ++r) q -= outk[r] != 0;
    while (q >= __popc(~taken[w])) q -= __popc(~taken[w]), ++w;
    id = w * 32 + __fns(~taken[w], 0, q + 1);
  }
  ids[(size_t)row * count + threadIdx.x] = id;
  vals[(size_t)row * count + threadIdx.x] = v;
}

// A CTA takes 256 PER ids of a row, a thread PER of them: VEC: four ids side by side at a time (16-byte loads of logits, 8-byte loads of counts); else one.  Their
// values stand in shared memory, where the few ids that a rule touches are worked out again by themselves.  What is done for every id is a load, a test of its
// count, a store, a load and a maximum, and its order is worked out only behind the threshold.  (With the rules and orders of all ids in registers, a division
// inlined for each, 64 rows of 151,936 ids took 36 us, both stages.)  Now 20.7 us, 59 MB or 9 us at the rate of a copy: bound by the chain of a CTA's phases -
// slot and masks, ids, rules, biases, threshold, list - with barriers between.  80 rows of 32,003 ids and 64 candidates 13.7 us, one row of 151,936 ids 6.5 us: two
// kernels of one CTA's latency each.
// Masked ids cost neither their logit nor their count.  An id at -inf is no candidate: it is one only where a row has fewer than `count` ids above -inf, and the
// second selection finds those by counting.
template <bool VEC, int PER>
__global__ void __launch_bounds__(PICK_THREADS, PICK_CTAS) pick_stage1_kernel(const __grid_constant__ PickArgs a) {
  pdl_launch();
  constexpr int W = VEC ? 4 : 1, N = PER / W, CHUNK = PICK_THREADS * PER;
  __shared__ PickShared sm;
  __shared__ __align__(16) float s_val[CHUNK];
  constexpr bool FINAL = PER == 16;                        // (the results' code in the other cost rows of many chunks 5 to 10 %)
  __shared__ uint64_t s_out[FINAL ? 64 : 1];
  __shared__ uint32_t s_taken[4];
  if (threadIdx.x == 0) sm.n = 0;
  if (FINAL && threadIdx.x < 4) s_taken[threadIdx.x] = 0;
  pdl_wait();
  __syncthreads();
  const int row = blockIdx.y, tid = threadIdx.x, base = blockIdx.x * CHUNK, ids_here = min(a.vocab - base, CHUNK);
  const int slot_in = a.row_slot != nullptr ? a.row_slot[row] : -1, slot = slot_in >= 0 && slot_in < a.n_slots ? slot_in : -1;
  const int mrow = a.mask != nullptr ? a.mask_row[row] : -1;
  const bool masked = mrow >= 0 && mrow < a.n_masks;
  const float* lr = a.logits + (size_t)row * a.ld + base;
  const uint16_t* cr = a.counts != nullptr && slot >= 0 ? a.counts + (size_t)slot * a.vocab + base : nullptr;
  const uint32_t* mr = a.mask + (size_t)(masked ? mrow : 0) * a.words + base / 32;
  // what the rules need is asked for before the ids' values
  const int* bid = a.bias_id != nullptr && slot >= 0 ? a.bias_id + (size_t)slot * a.n_bias : nullptr;
  const int nb = bid != nullptr ? a.n_bias : 0, window = a.first != nullptr && cr != nullptr ? a.first[row] : row;
  const int bias0 = tid < nb ? bid[tid] : -1, fed0 = a.first != nullptr && tid <= row ? a.fed[row - tid] : -1;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  if (cr != nullptr) rep = a.penalties[3 * slot], freq = a.penalties[3 * slot + 1], pres = a.penalties[3 * slot + 2];
  // which of the thread's ids may be taken: of ids (i * 256 + tid) W .. + W - 1, bits i W ..
  uint32_t ok = 0, touched = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * PICK_THREADS + tid) * W;
    uint32_t w = at < ids_here ? (1u << W) - 1 : 0u;
    if (masked && w != 0) w &= mr[at >> 5] >> (at & 31);
    ok |= w << (i * W);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * PICK_THREADS + tid) * W;
    const uint32_t mine = ok >> (i * W) & ((1u << W) - 1);
    if constexpr (VEC) {
      float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      uint2 c = make_uint2(0u, 0u);
      if (mine != 0) {
        v = *reinterpret_cast<const float4*>(lr + at);
        if (cr != nullptr) c = *reinterpret_cast<const uint2*>(cr + at);
      }
      if (masked) {
        if (!(mine & 1)) v.x = -INFINITY;
        if (!(mine & 2)) v.y = -INFINITY;
        if (!(mine & 4)) v.z = -INFINITY;
        if (!(mine & 8)) v.w = -INFINITY;
      }
      if ((c.x | c.y) != 0)
        touched |= ((c.x & 0xFFFFu ? 1u : 0u) | (c.x >> 16 ? 2u : 0u) | (c.y & 0xFFFFu ? 4u : 0u) | (c.y >> 16 ? 8u : 0u)) << (i * W);
      *reinterpret_cast<float4*>(s_val + at) = v;
    } else {
      const float v = mine ? lr[at] : -INFINITY;
      if (mine && cr != nullptr && cr[at] != 0) touched |= 1u << i;
      s_val[at] = v;
    }
  }
  // two at a time: their counts come from L2 once more
  while (touched != 0) {
    const int i = __ffs(touched) - 1, rest = touched & (touched - 1), k = rest != 0 ? __ffs(rest) - 1 : i;
    touched = rest & (rest - 1);
    const int at = (i / W * PICK_THREADS + tid) * W + i % W, to = (k / W * PICK_THREADS + tid) * W + k % W;
    const uint32_t word = cr[at], other = cr[to];
    const float v = s_val[at], u = s_val[to];
    if (v != -INFINITY) s_val[at] = pick_rules(v, word, 0, rep, freq, pres);                       // at -inf it stays, and a masked id is there
    if (k != i && u != -INFINITY) s_val[to] = pick_rules(u, other, 0, rep, freq, pres);
  }
  const int r0 = min(max(window, 0), row) + 1;             // the row's drafts: rows r0 .. row
  // Ids of the chunk with a bias or among the drafts are listed, with their places among the slot's biases (drafts: behind those).
  auto take = [&](int id, uint32_t place) {
    if (id < base || id - base >= ids_here) return;
    const int at = atomicAdd(&sm.n, 1);
    if (at < PICK_LIST) sm.list[at] = (uint64_t)id << 32 | place;
  };
  take(bias0, tid);
  if (row - tid >= r0) take(fed0, PICK_MAX_BIAS);
  for (int e = tid + PICK_THREADS; e < nb; e += PICK_THREADS) take(bid[e], e);
  for (int r = row - tid - PICK_THREADS; r >= r0; r -= PICK_THREADS) take(a.fed[r], PICK_MAX_BIAS);
  __syncthreads();
  const int listed = sm.n;
  if (listed > 0) {
    // Each such id again, with its drafts and biases; the first of an id adds up all of it in the order of the places.
    const float* bval = a.bias_val + (size_t)slot * a.n_bias;
    auto again = [&](int id, auto biases) {
      const int at = id - base;
      if (masked && !(mr[at >> 5] >> (at & 31) & 1)) return;
      uint32_t drafts = 0;
      for (int r = r0; r <= row; ++r) drafts += a.fed[r] == id;
      const float v = pick_rules(lr[at], cr != nullptr ? cr[at] : 0u, drafts, rep, freq, pres);
      float sum = 0.f;
      const bool any = biases(sum);
      s_val[at] = any ? __fadd_rn(v, sum) : v;
    };
    if (listed <= PICK_LIST) {
      for (int l = tid; l < listed; l += PICK_THREADS) {
        const uint64_t own = sm.list[l];
        const int id = (int)(own >> 32);
        uint64_t next = ~0ull;                             // the id's next place
        bool first = true;
        for (int j = 0; j < listed; ++j) {
          const uint64_t other = sm.list[j];
          if ((int)(other >> 32) != id) continue;
          if (other < own) first = false;
          else if (other > own) next = min(next, other);
        }
        if (!first) continue;                              // (a draft given twice: each the same)
        again(id, [&](float& sum) {
          uint32_t place = (uint32_t)own;
          if (place >= PICK_MAX_BIAS) return false;
          sum = bval[place];
          for (uint64_t to = next; to != ~0ull && (uint32_t)to < PICK_MAX_BIAS;) {
            place = (uint32_t)to;
            sum = __fadd_rn(sum, bval[place]);
            to = ~0ull;
            for (int j = 0; j < listed; ++j)
              if ((int)(sm.list[j] >> 32) == id && (uint32_t)sm.list[j] > place) to = min(to, sm.list[j]);
          }
          return true;
        });
      }
    } else {
      // more than the list holds: each for itself, an id more than once the same each time
      for (int l = tid; l < nb + row - r0 + 1; l += PICK_THREADS) {
        const int id = l < nb ? bid[l] : a.fed[r0 + l - nb];
        if (id < base || id - base >= ids_here) continue;
        again(id, [&](float& sum) {
          bool any = false;
          for (int f = 0; f < nb; ++f)
            if (bid[f] == id) sum = any ? __fadd_rn(sum, bval[f]) : bval[f], any = true;
          return any;
        });
      }
    }
    __syncthreads();
  }
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int at = (i * PICK_THREADS + tid) * W;
    if constexpr (VEC) {
      const float4 v = *reinterpret_cast<const float4*>(s_val + at);
      top = pick_max(top, pick_max(pick_max(v.x, v.y), pick_max(v.z, v.w)));
    } else {
      top = pick_max(top, s_val[at]);
    }
  }
  pick_select(top != -INFINITY ? pick_order(top) : 0u,
              [&](uint32_t least, auto f) {
                // from the lowest finite value on where all may pass, else -inf would be looked at one by one (a NaN: the values say nothing yet)
                const float lowest = -3.402823466e+38f, from = least < pick_order(lowest) ? lowest : pick_value(least);
                uint32_t hits = 0;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                  const int at = (i * PICK_THREADS + tid) * W;
                  if constexpr (VEC) {
                    const float4 v = *reinterpret_cast<const float4*>(s_val + at);
                    hits |= ((v.x < from ? 0u : 1u) | (v.y < from ? 0u : 2u) | (v.z < from ? 0u : 4u) | (v.w < from ? 0u : 8u)) << (i * W);
                  } else {
                    hits |= (s_val[at] < from ? 0u : 1u) << i;
                  }
                }
                while (hits != 0) {
                  const int i = __ffs(hits) - 1, at = (i / W * PICK_THREADS + tid) * W + i % W;
                  hits &= hits - 1;
                  const float v = s_val[at];
                  const uint32_t order = pick_order(v);
                  if (v != -INFINITY && order >= least) f(pick_key(order, base + at));
                }
              },
              a.count, FINAL && a.ids != nullptr ? s_out : a.cand + (size_t)row * a.nchunks * a.count + blockIdx.x, a.nchunks, sm);
  if (FINAL && a.ids != nullptr) {
    __syncthreads();
    pick_finish(s_out, s_taken, row, a.count, a.ids, a.vals);
  }
}

// total <= PICK_THREADS * 16 candidates a row, the chunks' best first, then their second best and so on: the best of all are then those of different threads.  (Chunk
// by chunk a few threads had most of them, the threshold let through more than the list holds, and four rows of 151,936 ids with 64 candidates took 37 us, then 11.)
__global__ void __launch_bounds__(PICK_THREADS) pick_stage2_kernel(const uint64_t* cand, int total, int count, int* __restrict__ ids, float* __restrict__ vals) {
  pdl_launch();
  pdl_wait();
  __shared__ PickShared sm;
  __shared__ uint64_t outk[64];
  __shared__ uint32_t taken[4];                            // of the ids below 128, those among the results
  if (threadIdx.x < 4) taken[threadIdx.x] = 0;
  const int row = blockIdx.x;
  const uint64_t* c = cand + (size_t)row * total;
  constexpr int PER = 16;
  uint64_t k[PER];
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int j = i * PICK_THREADS + threadIdx.x;
    k[i] = j < total ? c[j] : 0;
    mine = max(mine, (uint32_t)(k[i] >> 32));
  }
  pick_select(mine,
              [&](uint32_t least, auto f) {
#pragma unroll
                for (int i = 0; i < PER; ++i)
                  if ((uint32_t)(k[i] >> 32) >= least) f(k[i]);
              },
              count, outk, 1, sm);
  __syncthreads();
  pick_finish(outk, taken, row, count, ids, vals);
}

}  // namespace rx

using namespace rx;

RX_API int rx_token_counts(void* counts, int n_slots, int vocab, const void* slots, const void* starts, const void* prompt, const void* tokens, int n_tokens, int n,
                           int* status, void* stream) {
  if (n < 1 || n > 65535 || n_slots < 1 || vocab < 1 || vocab > (1 << 30) || n_tokens < 0 || n_tokens > (1 << 30)) return (int)cudaErrorInvalidValue;
  // As many slices as give every SM at most one CTA, but no more than shared memory asks for where that is not enough: one history of 151,936 ids in 75 slices 2.4 us, in
  // two 4.7 us; 64 histories in two slices each 6.6 us, in three - more CTAs than SMs - 8.2 us.  Slices of whole 16-byte words and whole halves of those.
  const int fewest = (vocab + CNT_MAX_SLICE - 1) / CNT_MAX_SLICE, wanted = 148 / n, most = (vocab + CNT_MIN_SLICE - 1) / CNT_MIN_SLICE;
  const int cut = wanted > most ? most : wanted, into = cut < fewest ? fewest : cut;
  const int slice = ((vocab + into - 1) / into + 15) & ~15, parts = (vocab + slice - 1) / slice;
  static bool configured[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !configured[dev]) {
    e = cudaFuncSetAttribute(token_counts_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, CNT_MAX_SLICE * 2 + 64);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) configured[dev] = true;
  }
  return (int)rx::launch(token_counts_kernel, dim3(parts, n), dim3(CNT_THREADS), (size_t)slice * 2, (cudaStream_t)stream, (uint16_t*)counts, (const int*)slots,
                         (const int*)starts, (const int*)prompt, (const int*)tokens, n_tokens, n_slots, vocab, slice, status);
}

RX_API int rx_token_counts_add(void* counts, int n_slots, int vocab, const void* slots, const void* tokens, int n, int in_prompt, int* status, void* stream) {
  if (n < 1 || n > (1 << 30) || n_slots < 1 || vocab < 1) return (int)cudaErrorInvalidValue;
  return (int)rx::launch(token_counts_add_kernel, dim3((n + 255) / 256), dim3(256), 0, (cudaStream_t)stream, (uint16_t*)counts, (const int*)slots, (const int*)tokens, n,
                         n_slots, vocab, in_prompt, status);
}

// scratch: rx_topk_scratch_bytes.  Any of counts (with penalties), bias_id (with bias_val), mask (with mask_row) and first (with fed) may be null.
RX_API int rx_topk_adjusted(const void* logits, long long ld, int rows, int vocab, int count, void* scratch, void* ids, void* vals, const void* row_slot,
                            const void* counts, const void* penalties, int n_slots, const void* bias_id, const void* bias_val, int n_bias, const void* mask,
                            const void* mask_row, int n_masks, const void* first, const void* fed, void* stream) {
  // Chunks of 4096 ids where all of them run at once: twice as many CTAs, each done sooner (with 8192: 80 rows of 32,003 ids 16.3 against 13.7 us, one row of 151,936
  // ids 7.2 against 6.6 us).  Else of 8192: half as many selections (64 rows of 151,936 ids 24.0 against 20.7 us; 54 rows, one candidate each, 19 against 20 us, though).
  const bool small = (long long)rows * ((vocab + 4095) / 4096) <= 148 * PICK_CTAS;
  const int nchunks = small ? (vocab + 4095) / 4096 : (vocab + 8191) / 8192;
  if (rows < 1 || rows > 65535 || vocab < 1 || count < 1 || count > 64 || count > vocab || (long long)nchunks * count > PICK_THREADS * 16 || ld < vocab || n_bias < 0 || n_bias > PICK_MAX_BIAS ||
      (first != nullptr && rows > PICK_MAX_WINDOW))
    return (int)cudaErrorInvalidValue;
  PickArgs a = {(const float*)logits, (const int*)row_slot, (const uint16_t*)counts, (const float*)penalties, (const int*)bias_id, (const float*)bias_val,
                (const uint32_t*)mask, (const int*)mask_row, (const int*)first, (const int*)fed, (uint64_t*)scratch, small && nchunks == 1 ? (int*)ids : nullptr, (float*)vals, ld, rows, vocab, n_slots, n_bias, n_masks,
                (vocab + 31) / 32, count, nchunks};
  // four ids at a time where every row of logits and counts begins on a 16- and an 8-byte boundary
  const bool vec = vocab % 4 == 0 && ld % 4 == 0 && ((uintptr_t)logits & 15) == 0 && ((uintptr_t)counts & 7) == 0;
  cudaStream_t st = (cudaStream_t)stream;
  const auto stage1 = small ? (vec ? pick_stage1_kernel<true, 16> : pick_stage1_kernel<false, 16>) : vec ? pick_stage1_kernel<true, 32> : pick_stage1_kernel<false, 32>;
  cudaError_t e = rx::launch(stage1, dim3(nchunks, rows), dim3(PICK_THREADS), 0, st, a);
  if (e != cudaSuccess || a.ids != nullptr) return (int)e;      // (2048 ids: 7.4 -> 5.5 us)
  return (int)rx::launch(pick_stage2_kernel, dim3(rows), dim3(PICK_THREADS), 0, st, (const uint64_t*)scratch, nchunks * count, count, (int*)ids, (float*)vals);
}
