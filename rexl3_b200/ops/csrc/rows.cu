// Row maps and block tables of a window or a prompt slice, from the requests' lengths (sm_100a).
//
// Request i holds have[i] cached tokens in table row seq[i] and feeds fed[i] more (none is allowed).  With starts = the exclusive sum of fed, its row
// starts[i] + j stands at position p = have[i] + j:
//     position p | slot table[seq][p / 64] * 64 + p % 64 | table row seq[i] | keys it sees p + 1 | common
// and the pages that the fed tokens begin, ceil((have + fed) / 64) - ceil(have / 64) of them, are taken from `free` in request order and written into the
// table.  common = how many leading table entries the request shares with the one before it that has rows, among the pages that hold cached tokens of both:
// what `attn_shared` groups rows by.
//
// All or nothing: every CTA checks all requests (a few KB) and works out their sums for itself, and a request that cannot be served leaves every
// output as it was.  (But a row whose table entry is no page - below 0, or of 2^25 and more, whose slots int32 cannot hold - gets slot -1, and the others are written.)
// Bound by latency (a chain of the loads of lengths, two scans of up to 1024 values, a table entry, a store), not by the 20 bytes a row
// that it writes: 64 requests of a row each 4.1 us, 23 prompts of 8000 rows together 4.9 us.  One launch: with `free_next` in the place of
// `free_at` a CTA would overwrite what another has yet to read, so the CTAs are one cluster that meets between the reading and the writing.  (One CTA instead
// of the eight: eight requests of up to five rows 3.3 against 3.1 us, 40 of them 4.9 against 4.0 us, 256 13.5 against 4.7 us.)
#include "common.cuh"

namespace rx {

constexpr int ROWS_PAGE = 64, ROWS_MAX_REQ = 1024, ROWS_THREADS = 512, ROWS_MAX_TABLE = 32768, ROWS_CLUSTER = 8;
constexpr int ROWS_WARPS = ROWS_THREADS / 32;

struct RowsArgs {
  const int *seq, *have, *fed, *free_ids, *free_at;
  int *table, *rows, *starts, *free_next, *status;
  int n, n_tables, width, cap, n_free;
};

// the last request of 0 .. n - 1 whose running sum `first` is at most x (requests without entries are passed over: their successor begins at the same place)
__device__ __forceinline__ int rows_owner(const int* first, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(ROWS_THREADS) window_rows_kernel(const RowsArgs a) {
  pdl_launch();
  __shared__ int s_seq[ROWS_MAX_REQ], s_have[ROWS_MAX_REQ], s_row[ROWS_MAX_REQ + 1], s_page[ROWS_MAX_REQ + 1], s_prev[ROWS_MAX_REQ];
  __shared__ uint32_t s_used[ROWS_MAX_TABLE / 32];
  __shared__ int s_sum[3][ROWS_WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = a.n;
  constexpr int ctas = ROWS_CLUSTER;
  const int cta = blockIdx.x;
  for (int i = tid; i < (a.n_tables + 31) / 32; i += ROWS_THREADS) s_used[i] = 0;
  pdl_wait();
  const int at0 = a.free_at != nullptr ? *a.free_at : 0;
  __syncthreads();
  // requests 2 tid and 2 tid + 1 are this thread's, so that one scan over the threads is one over the requests
  bool bad = at0 < 0;
  int fed[2], need[2], has[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = 2 * tid + u;
    fed[u] = need[u] = 0, has[u] = -1;
    if (i >= n) continue;
    const int seq = a.seq[i], have = a.have[i], f = a.fed[i];
    s_seq[i] = seq, s_have[i] = have;
    const long long end = (long long)have + f;
    if (seq < 0 || seq >= a.n_tables || have < 0 || f < 0 || f > a.cap || end > (long long)a.width * ROWS_PAGE) { bad = true; continue; }
    if (atomicOr(&s_used[seq >> 5], 1u << (seq & 31)) >> (seq & 31) & 1) bad = true;      // a table row twice
    fed[u] = f;
    if (f > 0) has[u] = i;
    if (a.free_at != nullptr) need[u] = (int)((end + ROWS_PAGE - 1) / ROWS_PAGE) - (have + ROWS_PAGE - 1) / ROWS_PAGE;
  }
  int row = fed[0] + fed[1], page = need[0] + need[1], last = max(has[0], has[1]);        // inclusive over the warp, then over the block
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int r = __shfl_up_sync(0xffffffffu, row, o), p = __shfl_up_sync(0xffffffffu, page, o), l = __shfl_up_sync(0xffffffffu, last, o);
    if (lane >= o) row += r, page += p, last = max(last, l);
  }
  if (lane == 31) s_sum[0][warp] = row, s_sum[1][warp] = page, s_sum[2][warp] = last;
  const int before_last = __shfl_up_sync(0xffffffffu, last, 1);
  bad = __syncthreads_or(bad);
  int rows_all = 0, pages_all = 0, l0 = lane > 0 ? before_last : -1;
  for (int w = 0; w < ROWS_WARPS; ++w) {
    if (w < warp) row += s_sum[0][w], page += s_sum[1][w], l0 = max(l0, s_sum[2][w]);
    rows_all += s_sum[0][w], pages_all += s_sum[1][w];
  }
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int i = 2 * tid + u;
    if (i >= n) continue;
    s_row[i] = u == 0 ? row - fed[1] - fed[0] : row - fed[1];
    s_page[i] = u == 0 ? page - need[1] - need[0] : page - need[1];
    s_prev[i] = u == 0 ? l0 : max(l0, has[0]);
  }
  if (tid == 0) s_row[n] = rows_all, s_page[n] = pages_all;
  bad = bad || rows_all > a.cap || (long long)at0 + pages_all > a.n_free;
  __syncthreads();
  cluster_sync();                                         // every CTA has read free_at
  if (bad) {
    if (cta == 0 && tid == 0) set_status(a.status, ST_BAD_ARG, 90, rows_all);
    return;
  }
  if (cta == 0) {
    for (int i = tid; i <= n; i += ROWS_THREADS) a.starts[i] = s_row[i];
    if (tid == 0 && a.free_next != nullptr) *a.free_next = at0 + pages_all;
  }
  const int gtid = cta * ROWS_THREADS + tid, all = ctas * ROWS_THREADS;
  for (int p = gtid; p < pages_all; p += all) {
    const int i = rows_owner(s_page, n, p);
    a.table[(size_t)s_seq[i] * a.width + (s_have[i] + ROWS_PAGE - 1) / ROWS_PAGE + (p - s_page[i])] = a.free_ids[at0 + p];
  }
  for (int r = gtid; r < rows_all; r += all) {
    const int i = rows_owner(s_row, n, r);
    const int seq = s_seq[i], have = s_have[i], pos = have + (r - s_row[i]), b = pos / ROWS_PAGE, held = (have + ROWS_PAGE - 1) / ROWS_PAGE;
    const int entry = a.free_at != nullptr && b >= held ? a.free_ids[at0 + s_page[i] + (b - held)] : a.table[(size_t)seq * a.width + b];
    const int id = entry <= 0x7FFFFFFF / ROWS_PAGE ? entry : -1;      // (a slot past int32)
    if (id < 0) set_status(a.status, ST_BAD_ARG, 91, r);
    a.rows[r] = pos;
    a.rows[(size_t)a.cap + r] = id < 0 ? -1 : id * ROWS_PAGE + pos % ROWS_PAGE;
    a.rows[2 * (size_t)a.cap + r] = seq;
    a.rows[3 * (size_t)a.cap + r] = pos + 1;
  }
  // a warp per request: entries that hold cached tokens are not among the ones that this call writes
  for (int i = cta * ROWS_WARPS + warp; i < n; i += ctas * ROWS_WARPS) {
    const int r0 = s_row[i], r1 = s_row[i + 1];
    if (r0 == r1) continue;
    const int j = s_prev[i];
    int common = 0;
    if (j >= 0) {
      const int most = (min(s_have[i], s_have[j]) + ROWS_PAGE - 1) / ROWS_PAGE;
      const int *x = a.table + (size_t)s_seq[i] * a.width, *y = a.table + (size_t)s_seq[j] * a.width;
      constexpr int U = 4;                                // entries in flight per lane and table
      common = most;
      for (int b = 0; b < most && common == most; b += 32 * U) {
        int d[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int e = b + 32 * u + lane;
          d[u] = e < most ? x[e] - y[e] : 0;
        }
#pragma unroll
        for (int u = U - 1; u >= 0; --u) {
          const unsigned differ = __ballot_sync(0xffffffffu, d[u] != 0);
          if (differ != 0) common = b + 32 * u + __ffs(differ) - 1;
        }
      }
    }
    for (int r = r0 + lane; r < r1; r += 32) a.rows[4 * (size_t)a.cap + r] = common;
  }
}

}  // namespace rx

using namespace rx;

// rows: int32 [5][cap].  free_at == nullptr: every page is in the table already.
RX_API int rx_window_rows(const void* seq, const void* have, const void* fed, int n, void* table, int n_tables, int width, const void* free_ids, int n_free,
                          const void* free_at, void* free_next, void* rows, int cap, void* starts, int* status, void* stream) {
  if (n < 1 || n > ROWS_MAX_REQ || n_tables < 1 || n_tables > ROWS_MAX_TABLE || width < 1 || width > (1 << 24) || cap < 0 || cap > (1 << 20) || n_free < 0)
    return (int)cudaErrorInvalidValue;
  if ((free_at == nullptr) != (free_next == nullptr) || ((free_ids == nullptr || free_at == nullptr) && n_free != 0)) return (int)cudaErrorInvalidValue;
  const RowsArgs a = {(const int*)seq, (const int*)have, (const int*)fed, (const int*)free_ids, (const int*)free_at, (int*)table, (int*)rows, (int*)starts,
                      (int*)free_next, status, n, n_tables, width, cap, n_free};
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ROWS_CLUSTER); cfg.blockDim = dim3(ROWS_THREADS); cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = ROWS_CLUSTER; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, window_rows_kernel, a);
}
