// Tables of a packed batch of sequences, built on the device from their lengths (or from a sorted segment index):
//   offsets[s] = sum_{q<s} len[q], index[i] = the segment of row i, position[i] = i - offsets[index[i]], bit i of `starts` = position[i] == 0,
// and, for rows kept in blocks of B rows of a shared store: request s owns blocks first[s] .. first[s] + ceil(len[s] / B) of the free list.
#include "tf_common.h"

namespace {

typedef long long ll;
typedef unsigned long long ull;

__device__ __forceinline__ ll seg_len(const ll* __restrict__ lengths, ll s, ll n_rows) { return min(max(lengths[s], 0ll), n_rows); }

// first segment whose END lies beyond row i: the segment that holds it (empty ones end where they begin and are passed over)
__device__ __forceinline__ ll seg_of_row(const ll* __restrict__ offsets, ll n_seg, ll i) {
  ll lo = 0, hi = n_seg;
  while (lo < hi) {
    const ll mid = (lo + hi) >> 1;
    if (offsets[mid + 1] <= i) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// exclusive sums of the lengths and of the block counts: one workgroup walks the list
__global__ void __launch_bounds__(1024) seg_sums_kernel(const ll* __restrict__ lengths, ll n_seg, ll n_rows, ll block_rows, ll* __restrict__ offsets,
                                                        ll* __restrict__ block_first) {
  __shared__ ll part[2][1024];
  const int t = threadIdx.x;
  ll base = 0, bbase = 0;
  for (ll s0 = 0; s0 < n_seg; s0 += 1024) {
    const ll s = s0 + t;
    const ll v = s < n_seg ? seg_len(lengths, s, n_rows) : 0;
    const ll b = block_rows ? (v + block_rows - 1) / block_rows : 0;
    part[0][t] = v;
    part[1][t] = b;
    __syncthreads();
    for (int o = 1; o < 1024; o <<= 1) {
      const ll p = t >= o ? part[0][t - o] : 0, q = t >= o ? part[1][t - o] : 0;
      __syncthreads();
      part[0][t] += p;
      part[1][t] += q;
      __syncthreads();
    }
    if (s < n_seg) {
      offsets[s] = min(base + part[0][t] - v, n_rows);
      if (block_rows) block_first[s] = bbase + part[1][t] - b;
    }
    base += part[0][1023];
    bbase += part[1][1023];
    __syncthreads();
  }
  if (t == 0) offsets[n_seg] = min(base, n_rows);
}

__global__ void __launch_bounds__(256) seg_rows_kernel(const ll* __restrict__ offsets, const int* __restrict__ table, ll n_seg, ll n_rows, ll block_rows,
                                                       ll max_blocks, ll* __restrict__ index, ll* __restrict__ position, ull* __restrict__ starts,
                                                       ll* __restrict__ slots) {
  const ll i = (ll)blockIdx.x * 256 + threadIdx.x;
  const bool in = i < n_rows;
  const ll s = in ? seg_of_row(offsets, n_seg, i) : n_seg;
  const bool ok = s < n_seg;
  const ll p = ok ? i - offsets[s] : -1;
  const ull bits = __ballot(p == 0);
  if (!in) return;
  if (index) index[i] = ok ? s : -1;
  if (position) position[i] = p;
  if (starts && (threadIdx.x & 63) == 0) starts[i >> 6] = bits;
  if (slots) {
    ll v = -1;
    if (ok && p / block_rows < max_blocks) {
      const int blk = table[s * max_blocks + p / block_rows];
      if (blk >= 0) v = blk * block_rows + p % block_rows;
    }
    slots[i] = v;
  }
}

__global__ void __launch_bounds__(256) seg_blocks_kernel(const ll* __restrict__ lengths, const ll* __restrict__ block_first, const int* __restrict__ free_blocks,
                                                         ll n_free, ll n_seg, ll n_rows, ll block_rows, ll max_blocks, int* __restrict__ table) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x;
  if (e >= n_seg * max_blocks) return;
  const ll s = e / max_blocks, c = e % max_blocks;
  const ll have = (seg_len(lengths, s, n_rows) + block_rows - 1) / block_rows, at = block_first[s] + c;
  table[e] = c < have && at < n_free ? free_blocks[at] : -1;
}

// first row of a sorted index that is >= s
__global__ void __launch_bounds__(256) seg_bounds_kernel(const ll* __restrict__ index, ll n_rows, ll n_seg, ll* __restrict__ offsets) {
  const ll s = (ll)blockIdx.x * 256 + threadIdx.x;
  if (s > n_seg) return;
  ll lo = 0, hi = n_rows;
  while (lo < hi) {
    const ll mid = (lo + hi) >> 1;
    if (index[mid] < s) lo = mid + 1; else hi = mid;
  }
  offsets[s] = lo;
}

__global__ void __launch_bounds__(256) seg_starts_kernel(const ll* __restrict__ index, ll n_rows, ll n_seg, ull* __restrict__ starts) {
  const ll i = (ll)blockIdx.x * 256 + threadIdx.x;
  const bool in = i < n_rows;
  const ll s = in ? index[i] : -1;
  const ull bits = __ballot(in && s >= 0 && s < n_seg && (i == 0 || index[i - 1] != s));
  if (in && (threadIdx.x & 63) == 0) starts[i >> 6] = bits;
}

inline bool grid_fits(ll n, ll per) { return (n + per - 1) / per < (1ll << 31); }

}  // namespace

extern "C" size_t tf_segment_workspace_words(int64_t n_segments, int64_t block_rows) {
  return block_rows > 0 && n_segments > 0 ? (size_t)n_segments : 0;
}

extern "C" int tf_segment_tables(const int64_t* lengths, int64_t n_segments, int64_t n_rows, int64_t* offsets, int64_t* index, int64_t* position,
                                 uint64_t* starts, int64_t block_rows, const int32_t* free_blocks, int64_t n_free, int64_t max_blocks,
                                 int32_t* block_table, int64_t* slots, int64_t* workspace, size_t workspace_words, tf_stream_t stream) {
  TF_REQUIRE(n_segments >= 0 && n_rows >= 0 && block_rows >= 0 && n_free >= 0 && max_blocks >= 0, TF_ESHAPE, "tf_segment_tables: negative size");
  TF_REQUIRE(grid_fits(n_rows, 256) && grid_fits(n_segments, 256), TF_ESHAPE, "tf_segment_tables: too many rows or segments");
  TF_REQUIRE(offsets && (n_segments == 0 || lengths), TF_EINVAL, "tf_segment_tables: null pointer");
  const bool blocks = block_rows > 0;
  TF_REQUIRE(blocks || (!block_table && !slots), TF_EINVAL, "tf_segment_tables: block outputs without a block size");
  if (blocks) {
    TF_REQUIRE(max_blocks == 0 || grid_fits(n_segments, 256 / (max_blocks < 256 ? max_blocks : 256)), TF_ESHAPE, "tf_segment_tables: block table too large");
    TF_REQUIRE(n_segments == 0 || max_blocks == 0 || n_segments < (1ll << 39) / max_blocks, TF_ESHAPE, "tf_segment_tables: block table too large");
    TF_REQUIRE((n_free == 0 || free_blocks) && (n_segments * max_blocks == 0 || block_table), TF_EINVAL, "tf_segment_tables: null block pointer");
    TF_REQUIRE(workspace_words >= tf_segment_workspace_words(n_segments, block_rows) && (n_segments == 0 || workspace), TF_ESHAPE,
               "tf_segment_tables: workspace too small");
  }
  hipStream_t st = (hipStream_t)stream;
  seg_sums_kernel<<<1, 1024, 0, st>>>((const ll*)lengths, n_segments, n_rows, block_rows, (ll*)offsets, (ll*)workspace);
  if (blocks && n_segments * max_blocks > 0)
    seg_blocks_kernel<<<(unsigned)((n_segments * max_blocks + 255) / 256), 256, 0, st>>>((const ll*)lengths, (const ll*)workspace, free_blocks, n_free, n_segments,
                                                                                       n_rows, block_rows, max_blocks, block_table);
  if (n_rows > 0 && (index || position || starts || slots))
    seg_rows_kernel<<<(unsigned)((n_rows + 255) / 256), 256, 0, st>>>((const ll*)offsets, block_table, n_segments, n_rows, block_rows, max_blocks, (ll*)index,
                                                                    (ll*)position, (ull*)starts, (ll*)slots);
  TF_LAUNCH_CHECK("tf_segment_tables");
  return TF_OK;
}

extern "C" int tf_segment_from_index(const int64_t* index, int64_t n_rows, int64_t n_segments, int64_t* offsets, uint64_t* starts, tf_stream_t stream) {
  TF_REQUIRE(n_segments >= 0 && n_rows >= 0, TF_ESHAPE, "tf_segment_from_index: negative size");
  TF_REQUIRE(grid_fits(n_rows, 256) && grid_fits(n_segments + 1, 256), TF_ESHAPE, "tf_segment_from_index: too many rows or segments");
  TF_REQUIRE(offsets && (n_rows == 0 || (index && starts)), TF_EINVAL, "tf_segment_from_index: null pointer");
  hipStream_t st = (hipStream_t)stream;
  seg_bounds_kernel<<<(unsigned)((n_segments + 1 + 255) / 256), 256, 0, st>>>((const ll*)index, n_rows, n_segments, (ll*)offsets);
  if (n_rows > 0) seg_starts_kernel<<<(unsigned)((n_rows + 255) / 256), 256, 0, st>>>((const ll*)index, n_rows, n_segments, (ull*)starts);
  TF_LAUNCH_CHECK("tf_segment_from_index");
  return TF_OK;
}
