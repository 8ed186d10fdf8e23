// Tables of a packed batch of sequences, built on the device from their lengths (or from a sorted segment index):
//   offsets[s] = sum_{q<s} len[q], index[i] = the segment of row i, position[i] = i - offsets[index[i]], bit i of `starts` = position[i] == 0,
// and, for rows kept in blocks of B rows of a shared store: segment s owns entries first[s] .. first[s] + ceil(len[s] / B) of the free list.
// Bound: the launch for a batch, the writes (8 bytes a row and table) for a frame.
#include "tf_common.h"

namespace {

typedef long long ll;
typedef unsigned long long ull;

// Up to SMALL segments every workgroup sums the lengths by itself and finds its rows' segments in LDS: ONE launch, where the sums' own would cost
// as much again (1024 segments, 130003 rows: 9.6 us of kernels in two, 7.7 in one).  More segments: sums, offsets, rows.
constexpr int SMALL = 2048;
constexpr int WAVE_ROWS = 1024;  // rows of a wave of the rows

__device__ __forceinline__ ll seg_len(const ll* __restrict__ lengths, ll s, ll n_rows) { return min(max(lengths[s], 0ll), n_rows); }

struct Blocks {
  ll rows, n_free, max_blocks;
  const int* free_blocks;
  int* table;
  ll* slots;
  int shift;  // log2(rows), or -1
};
__device__ __forceinline__ ll blocks_of(const Blocks& b, ll n) { return b.shift >= 0 ? (n + b.rows - 1) >> b.shift : (n + b.rows - 1) / b.rows; }
__device__ __forceinline__ ll slot_of(const Blocks& b, ll first, ll pos) {
  const ll c = b.shift >= 0 ? pos >> b.shift : pos / b.rows;
  if (c >= b.max_blocks || first + c >= b.n_free) return -1;
  const ll blk = b.free_blocks[first + c];
  return blk < 0 ? -1 : blk * b.rows + (pos - c * b.rows);
}

__device__ __forceinline__ ll wave_inclusive(ll v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const ll p = __shfl_up(v, o);
    if (lane >= o) v += p;
  }
  return v;
}
// exclusive sums over the workgroup's threads; `total` of all of them
template <int WAVES>
__device__ __forceinline__ ll block_exclusive(ll v, ll* part, ll& total) {
  const int wave = threadIdx.x >> 6;
  const ll in = wave_inclusive(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) part[wave] = in;
  __syncthreads();
  ll before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < WAVES; ++w) {
    if (w < wave) before += part[w];
    total += part[w];
  }
  return before + in - v;
}

__global__ void __launch_bounds__(256) seg_small_kernel(const ll* __restrict__ lengths, int n_seg, ll n_rows, ll rows_per_block, ll* __restrict__ offsets,
                                                        ll* __restrict__ index, ll* __restrict__ position, ull* __restrict__ starts, Blocks b) {
  __shared__ ll off[SMALL + 1], first[SMALL], part[4];
  constexpr int PER = SMALL / 256;
  const int t = threadIdx.x;
  ll v[PER], sum = 0, bsum = 0, total, btotal;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int s = t * PER + k;
    v[k] = s < n_seg ? seg_len(lengths, s, n_rows) : 0;
    sum += v[k];
    if (b.rows) bsum += blocks_of(b, v[k]);
  }
  ll at = block_exclusive<4>(sum, part, total), bat = b.rows ? block_exclusive<4>(bsum, part, btotal) : 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int s = t * PER + k;
    if (s < n_seg) {
      off[s] = min(at, n_rows);
      if (b.rows) first[s] = bat;
    }
    at += v[k];
    if (b.rows) bat += blocks_of(b, v[k]);
  }
  if (t == 0) off[n_seg] = min(total, n_rows);
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = t; s <= n_seg; s += 256) offsets[s] = off[s];
  if (b.table) {
    const ll n = n_seg * b.max_blocks;
    for (ll e = (ll)blockIdx.x * 256 + t; e < n; e += (ll)gridDim.x * 256) {
      const int s = n < (1ll << 31) ? (int)((unsigned)e / (unsigned)b.max_blocks) : (int)(e / b.max_blocks);
      const ll c = e - s * b.max_blocks;
      b.table[e] = c < blocks_of(b, seg_len(lengths, s, n_rows)) && first[s] + c < b.n_free ? b.free_blocks[first[s] + c] : -1;
    }
  }
  if (!starts) return;
  const ll r1 = min(n_rows, (blockIdx.x + 1) * rows_per_block), end = off[n_seg];
  for (ll base = blockIdx.x * rows_per_block; base < r1; base += 256) {
    const ll i = base + t;
    // the first segment whose END lies beyond row i: the one that holds it (empty ones end where they begin and are passed over)
    int lo = 0, hi = n_seg;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (off[mid + 1] <= i) lo = mid + 1; else hi = mid;
    }
    const bool ok = i < end;
    const ll p = ok ? i - off[lo] : -1;
    const ull bits = __ballot(p == 0);
    if (i < r1) {
      if ((t & 63) == 0) starts[i >> 6] = bits;
      if (index) index[i] = ok ? lo : -1;
      if (position) position[i] = p;
      if (b.slots) b.slots[i] = ok ? slot_of(b, first[lo], p) : -1;
    }
  }
}

// PER lengths a thread: 2 up to a million segments (640000: sums and offsets 20 us, 27 with 8), 16 beyond, where every workgroup adds up the sums of
// all before it.
// sums of a workgroup's lengths (and of their block counts); the start bits cleared.  A sum counts for no more than all rows (all free blocks): what lies
// behind is cut at the same place, and 2^31 segments of up to 2^39 rows sum to 2^58 at most.
template <int PER>
__global__ void __launch_bounds__(256) seg_sums_kernel(const ll* __restrict__ lengths, ll n_seg, ll n_rows, Blocks b, ll* __restrict__ sums,
                                                       ull* __restrict__ starts, ll n_words) {
  __shared__ ll part[4];
  const ll s0 = (ll)blockIdx.x * (256 * PER);
  ll sum = 0, bsum = 0, total;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const ll s = s0 + k * 256 + threadIdx.x;
    if (s < n_seg) {
      const ll v = seg_len(lengths, s, n_rows);
      sum += v;
      if (b.rows) bsum += blocks_of(b, v);
    }
  }
  block_exclusive<4>(sum, part, total);
  if (threadIdx.x == 0) sums[2 * blockIdx.x] = min(total, n_rows);
  if (b.rows) block_exclusive<4>(bsum, part, total);
  if (threadIdx.x == 0) sums[2 * blockIdx.x + 1] = b.rows ? min(total, b.n_free) : 0;
  if (starts)
    for (ll w = (ll)blockIdx.x * 256 + threadIdx.x; w < n_words; w += (ll)gridDim.x * 256) starts[w] = 0;
}

// offsets from the sums; every segment with rows marks its first one: the start bit, and its number in index
template <int PER>
__global__ void __launch_bounds__(256) seg_offsets_kernel(const ll* __restrict__ lengths, ll n_seg, ll n_rows, Blocks b, const ll* __restrict__ sums,
                                                          ll* __restrict__ offsets, ll* __restrict__ block_first, ll* __restrict__ index, ull* __restrict__ starts) {
  __shared__ ll part[4];
  ll base = 0, bbase = 0, total;
  for (ll c = threadIdx.x; c < blockIdx.x; c += 256) {
    base += sums[2 * c];
    bbase += sums[2 * c + 1];
  }
  block_exclusive<4>(base, part, total);
  base = total;
  block_exclusive<4>(bbase, part, total);
  bbase = total;
  ll v[PER], sum = 0, bsum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const ll s = ((ll)blockIdx.x * 256 + threadIdx.x) * PER + k;
    v[k] = s < n_seg ? seg_len(lengths, s, n_rows) : 0;
    sum += v[k];
    if (b.rows) bsum += blocks_of(b, v[k]);
  }
  base += block_exclusive<4>(sum, part, total);
  if (b.rows) bbase += block_exclusive<4>(bsum, part, total);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const ll s = ((ll)blockIdx.x * 256 + threadIdx.x) * PER + k, at = min(base, n_rows);
    if (s < n_seg) {
      offsets[s] = at;
      if (b.rows) block_first[s] = bbase;
      if (s == n_seg - 1) offsets[n_seg] = min(at + v[k], n_rows);
      if (starts && v[k] > 0 && at < n_rows) {
        atomicOr(starts + (at >> 6), 1ull << (at & 63));
        if (index) index[at] = s;
      }
    }
    base += v[k];
    if (b.rows) bbase += blocks_of(b, v[k]);
  }
}

// the segment that holds row i < offsets[n_seg], by all lanes: 64 probes a round
__device__ __forceinline__ ll wave_seg_of(const ll* __restrict__ offsets, ll n_seg, ll i) {
  const int lane = threadIdx.x & 63;
  ll lo = 0, n = n_seg;
  while (n > 1) {
    const ll step = (n + 63) >> 6, at = lo + lane * step + step - 1;
    const ull hit = __ballot(at >= lo + n - 1 || offsets[at + 1] > i);
    const int f = __ffsll((long long)hit) - 1;
    lo += f * step;
    n = min(step, n - f * step);
  }
  return lo;
}

// Every row from the start bits: a row belongs to the last start at or before it, among the wave's 128 rows or carried from before.  A lane has two rows
// side by side, stored as one piece of 16 bytes (33.3 million rows, 640000 segments, two tables: 91 us; 180 with a row and 8 bytes a lane).
typedef ll ll2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void put2(ll* p, ll i, ll n, bool pair, ll a, ll b) {
  if (pair && i + 1 < n) {
    __builtin_nontemporal_store(ll2{a, b}, reinterpret_cast<ll2*>(p + i));
  } else {
    if (i < n) p[i] = a;
    if (i + 1 < n) p[i + 1] = b;
  }
}
__global__ void __launch_bounds__(256) seg_rows_kernel(const ll* __restrict__ offsets, const ll* __restrict__ block_first, ll n_seg, ll n_rows,
                                                       const ull* __restrict__ starts, ll* index, ll* __restrict__ position, Blocks b, bool pair) {
  constexpr int N = WAVE_ROWS / 128;
  const int lane = threadIdx.x & 63;
  const ll row0 = ((ll)blockIdx.x * 4 + (threadIdx.x >> 6)) * WAVE_ROWS, end = offsets[n_seg], words = (n_rows + 63) >> 6;
  if (row0 >= n_rows) return;
  // the two start bits of the lane's rows in each of the wave's stretches of 128, and the segments that begin there
  unsigned two[N];
  ll s0[N], s1[N];
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const ll w = (row0 >> 6) + 2 * k + (lane >> 5);
    two[k] = w < words ? (unsigned)(starts[w] >> (2 * lane & 63)) & 3 : 0;
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const ll i = row0 + 128 * k + 2 * lane;
    s0[k] = index && (two[k] & 1) ? index[i] : 0;
    s1[k] = index && (two[k] & 2) ? index[i + 1] : 0;
  }
  ll cseg = -1, cstart = 0;
  if (!(__builtin_amdgcn_readfirstlane(two[0]) & 1) && row0 < end) {
    cseg = wave_seg_of(offsets, n_seg, row0);
    cstart = offsets[cseg];
  }
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const ll base = row0 + 128 * k, i = base + 2 * lane;
    const ull any = __ballot(two[k] != 0), odd = __ballot(two[k] & 2), before = any & ((1ull << lane) - 1);
    const ll mine = two[k] & 2 ? s1[k] : s0[k];
    // the last start in front of the lane's rows, and the last of all
    const int src = before ? 63 - __clzll((long long)before) : 0, top = any ? 63 - __clzll((long long)any) : 0;
    const ll got = __shfl(mine, src), last = __shfl(mine, top);
    const ll ps = before ? got : cseg, pstart = before ? base + 2 * src + (ll)(odd >> src & 1) : cstart;
    const ll sa = two[k] & 1 ? s0[k] : ps, pa = two[k] & 1 ? 0 : i - pstart;
    const ll sb = two[k] & 2 ? s1[k] : sa, pb = two[k] & 2 ? 0 : pa + 1;
    if (any) {
      cseg = last;
      cstart = base + 2 * top + (ll)(odd >> top & 1);
    }
    const bool oka = i < end, okb = i + 1 < end;
    if (index) put2(index, i, n_rows, pair, oka ? sa : -1, okb ? sb : -1);
    if (position) put2(position, i, n_rows, pair, oka ? pa : -1, okb ? pb : -1);
    if (b.slots) put2(b.slots, i, n_rows, pair, oka ? slot_of(b, block_first[sa], pa) : -1, okb ? slot_of(b, block_first[sb], pb) : -1);
  }
}

__global__ void __launch_bounds__(256) seg_blocks_kernel(const ll* __restrict__ lengths, const ll* __restrict__ block_first, ll n_seg, ll n_rows, Blocks b) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x, n = n_seg * b.max_blocks;
  if (e >= n) return;
  const ll s = n < (1ll << 31) ? (ll)((unsigned)e / (unsigned)b.max_blocks) : e / b.max_blocks, c = e - s * b.max_blocks, at = block_first[s] + c;
  b.table[e] = c < blocks_of(b, seg_len(lengths, s, n_rows)) && at < b.n_free ? b.free_blocks[at] : -1;
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
inline int per_of(ll n_seg) { return n_seg <= (1 << 20) ? 2 : 16; }
inline ll chunks_of(ll n_seg) { return (n_seg + 256 * per_of(n_seg) - 1) / (256 * per_of(n_seg)); }

}  // namespace

extern "C" size_t tf_segment_workspace_words(int64_t n_segments, int64_t block_rows) {
  if (n_segments <= SMALL) return 0;
  return 2 * (size_t)chunks_of(n_segments) + (block_rows > 0 ? (size_t)n_segments : 0);
}

extern "C" int tf_segment_tables(const int64_t* lengths, int64_t n_segments, int64_t n_rows, int64_t* offsets, int64_t* index, int64_t* position,
                                 uint64_t* starts, int64_t block_rows, const int32_t* free_blocks, int64_t n_free, int64_t max_blocks,
                                 int32_t* block_table, int64_t* slots, int64_t* workspace, size_t workspace_words, tf_stream_t stream) {
  TF_REQUIRE(n_segments >= 0 && n_rows >= 0 && block_rows >= 0 && n_free >= 0 && max_blocks >= 0, TF_ESHAPE, "tf_segment_tables: negative size");
  TF_REQUIRE(grid_fits(n_rows, 256) && grid_fits(n_segments, 256), TF_ESHAPE, "tf_segment_tables: too many rows or segments");
  TF_REQUIRE(offsets && (n_segments == 0 || lengths), TF_EINVAL, "tf_segment_tables: null pointer");
  TF_REQUIRE(n_rows == 0 || starts || (!index && !position && !slots), TF_EINVAL, "tf_segment_tables: tables of rows need starts");
  const bool blocks = block_rows > 0;
  TF_REQUIRE(blocks || (!block_table && !slots), TF_EINVAL, "tf_segment_tables: block outputs without a block size");
  if (blocks) {
    TF_REQUIRE(n_segments == 0 || max_blocks == 0 || n_segments < (1ll << 38) / max_blocks, TF_ESHAPE, "tf_segment_tables: block table too large");
    TF_REQUIRE(block_rows < (1ll << 31), TF_ESHAPE, "tf_segment_tables: blocks too large");
    TF_REQUIRE((n_free == 0 || free_blocks) && (n_segments * max_blocks == 0 || block_table), TF_EINVAL, "tf_segment_tables: null block pointer");
    TF_REQUIRE(!slots || index, TF_EINVAL, "tf_segment_tables: slots need an index");
  }
  TF_REQUIRE(workspace_words >= tf_segment_workspace_words(n_segments, block_rows) && (workspace || !tf_segment_workspace_words(n_segments, block_rows)),
             TF_ESHAPE, "tf_segment_tables: workspace too small");
  hipStream_t st = (hipStream_t)stream;
  const ll cells = blocks ? n_segments * max_blocks : 0;
  Blocks b = {block_rows, n_free, max_blocks, free_blocks, cells ? block_table : nullptr, (ll*)slots, -1};
  if (blocks && (block_rows & (block_rows - 1)) == 0)
    for (b.shift = 0; (1ll << b.shift) < block_rows;) ++b.shift;
  if (n_segments <= SMALL) {
    // a workgroup's rows: enough of them to be worth its sums, few enough to fill the card
    const ll per = n_rows < (1ll << 20) ? 1024 : 8192;
    ll grid = starts ? (n_rows + per - 1) / per : 0;
    if (cells && grid < (cells + 1023) / 1024) grid = (cells + 1023) / 1024 < 2048 ? (cells + 1023) / 1024 : 2048;
    TF_REQUIRE(grid < (1ll << 31), TF_ESHAPE, "tf_segment_tables: too many rows");
    seg_small_kernel<<<(unsigned)(grid ? grid : 1), 256, 0, st>>>((const ll*)lengths, (int)n_segments, n_rows, per, (ll*)offsets, (ll*)index, (ll*)position,
                                                                (ull*)starts, b);
  } else {
    ll* sums = (ll*)workspace;
    ll* first = sums + 2 * chunks_of(n_segments);
    const unsigned grid = (unsigned)chunks_of(n_segments);
    const bool pair = (((size_t)index | (size_t)position | (size_t)slots) & 15) == 0;
    const ll words = starts ? (n_rows + 63) >> 6 : 0;
#define SUMS(PER)                                                                                                                            \
  seg_sums_kernel<PER><<<grid, 256, 0, st>>>((const ll*)lengths, n_segments, n_rows, b, sums, (ull*)starts, words);                           \
  seg_offsets_kernel<PER><<<grid, 256, 0, st>>>((const ll*)lengths, n_segments, n_rows, b, sums, (ll*)offsets, first, (ll*)index, (ull*)starts)
    if (per_of(n_segments) == 2) {
      SUMS(2);
    } else {
      SUMS(16);
    }
#undef SUMS
    if (cells) seg_blocks_kernel<<<(unsigned)((cells + 255) / 256), 256, 0, st>>>((const ll*)lengths, first, n_segments, n_rows, b);
    if (n_rows > 0 && (index || position))
      seg_rows_kernel<<<(unsigned)((n_rows + 4 * WAVE_ROWS - 1) / (4 * WAVE_ROWS)), 256, 0, st>>>((const ll*)offsets, first, n_segments, n_rows, (const ull*)starts,
                                                                                              (ll*)index, (ll*)position, b, pair);
  }
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
