// Forward pass of the gated linear recurrence over a packed batch (scan_tile.h has the decomposition).
//   TF_GATE_DECAY: a = g, b = x;   TF_GATE_LOG: a = exp(g), b = x;   TF_GATE_ALPHA: a = 1 - g, b = g x (compositing).
#include "scan_tile.h"

using namespace tfscan;

namespace {

// No kernel here may spill vector registers (no_spills.py ends the build; the bounds below are the tightest that none does).  Scalar registers are spilled in
// all of them, 75 to 106, into lanes of vector registers.  Measured: 65536 x 1024 bf16 with a bf16 gate for each channel, one sequence, 134 us (403 MB, 3.0
// TB/s): a tile of 15 us spends 4.6 on its loads, 1.5 on its own map, 5.8 on its place in the chain and 2.5 on its stores, and two
// tiles to a CU do not fill each other's pauses.  Tried and slower: 16 rows a lane (155 us, registers), 4 rows (180), workgroups that stay and touch their next
// tile's lines ahead (161), the next tile's rows held in registers (they spill).
template <typename XT, typename GT, int V, bool SHARED, bool WIDE>
__global__ void __launch_bounds__(512, SHARED || (WIDE && sizeof(XT) == 2) ? 4 : 3)
    scan_fwd_kernel(ScanArgs p, XT* __restrict__ y, float* __restrict__ final, float* __restrict__ carry) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  __shared__ unsigned s_ticket;
  __shared__ int s_closed[8], s_opened;
  constexpr int AV = SHARED ? 1 : V;
  const int nw = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  float *sA = smem, *sB = smem + nw * p.W;
  char* buf = reinterpret_cast<char*>(smem + (2 * nw * p.W + 3 & ~3)) + wave * p.narrow;
  const ll lo = max(p.offsets[0], 0ll), hi = min(p.offsets[p.n_seg], p.n_rows);
  int slab;
  const int q = take_job(p, &s_ticket, slab);
  if (slab < 0) {
    empty_segments(p, (ll)q * nw + wave, p.h0, final);
    return;
  }
  const int cl = WIDE ? lane : lane & (p.CL - 1), rl = WIDE ? 0 : lane / p.CL, RL = WIDE ? 1 : 64 / p.CL, T = nw * RL * K;
  const Lane<V, SHARED> l(p, slab, cl);
  const Rows<WIDE> r(p, (ll)q * T + (wave * RL + rl) * K, T, lo, hi);
  const ll t0 = (ll)(p.reverse ? p.tiles - 1 - q : q) * T;  // the tile's lowest row, and its wave's
  const ll w0 = t0 + (ll)(p.reverse ? nw - 1 - wave : wave) * RL * K;
  const int block = p.reverse ? RL - 1 - rl : rl;
  const bool full = t0 >= lo && t0 + T <= hi, turned = !WIDE && p.narrow && full;
  Raw<XT, V> x[K];
  Raw<GT, AV> g[K];
  unsigned first, last;
  if (turned) {
    Turn<XT, V> tx(p.D, RL);
    Turn<GT, AV> tg(p.G, RL);
    tx.load(static_cast<const XT*>(p.x) + w0 * p.D);
    tg.load(static_cast<const GT*>(p.gate) + w0 * p.G);
    r.bits(p, hi, first, last);
    tx.to_rows(buf, p.D, block, l.c, p.reverse, x);
    tg.to_rows(buf, p.G, block, l.g, p.reverse, g);
  } else {
    direct_rows<XT, V, WIDE>(static_cast<const XT*>(p.x), p.ld_x, r, l.c, full, x);
    direct_rows<GT, AV, WIDE>(static_cast<const GT*>(p.gate), p.ld_gate, r, l.g, full, g);
    r.bits(p, hi, first, last);
  }
  // a row's a and b: in place of g and x where those are fp32 (40001 x 512 in two sequences: 10 us less than with both computed in either pass), from
  // the packed values each time where they are not
  constexpr bool WHOLE = sizeof(XT) == 4;
  const bool alpha = p.form == TF_GATE_ALPHA;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    gates_kept<GT, AV>(g[k], p.form);
    if (WHOLE && alpha) {
#pragma unroll
      for (int v = 0; v < V; ++v) x[k].w[v] = __builtin_bit_cast(unsigned, x[k][v] * g[k][AV == 1 ? 0 : v]);
#pragma unroll
      for (int v = 0; v < AV; ++v) g[k].w[v] = __builtin_bit_cast(unsigned, 1.f - g[k][v]);
    }
  }
  const float s1 = alpha ? -1.f : 1.f, s0 = alpha ? 1.f : 0.f;
  auto terms = [&](int k, float (&a)[AV], float (&b)[V]) {
    gates_of<GT, AV>(g[k], p.form, a);
#pragma unroll
    for (int v = 0; v < V; ++v) b[v] = !WHOLE && alpha ? a[AV == 1 ? 0 : v] * x[k][v] : x[k][v];
    if (!WHOLE) {
#pragma unroll
      for (int v = 0; v < AV; ++v) a[v] = fmaf(a[v], s1, s0);
    }
  };
  // the states that segments begin from (0 where there is no h0), for all of a lane's rows at once: b + a h0 in the place of b, which is then the first row's
  // state.  The product with a 0 stays: an infinite decay gives here what it gives in the other kernels and in the backward pass.
  constexpr bool JOINED = !WIDE && WHOLE;
  const float* h0 = p.h0;
  if (JOINED && __any(first)) {
    float s[K][V] = {};
    if (h0) {
      int seg[K];
      segs_of<WIDE>(p, r, first, seg);
      states_of<V>(p, h0, seg, l.c, s);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) s[k][v] = seg[k] >= 0 ? s[k][v] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int v = 0; v < V; ++v)
        x[k].w[v] = __builtin_bit_cast(unsigned, first >> k & 1 ? fmaf(g[k][AV == 1 ? 0 : v], s[k][v], x[k][v]) : x[k][v]);
  }
  // a first row begins from h0 (or 0), a row of no segment from 0: it holds b = 0 and leaves 0
  unsigned cut = first | (~r.valid & ((1u << K) - 1));
  float A[AV], B[V], eA[AV], eB[V];
  bool closed = cut != 0, eclosed;
#pragma unroll
  for (int v = 0; v < AV; ++v) A[v] = 1.f;
#pragma unroll
  for (int v = 0; v < V; ++v) B[v] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!JOINED) cut_at<V, WIDE>(p, k, cut, first, h0, r.p0 + k * r.step, l.c, B);
    float a[AV], b[V];
    terms(k, a, b);
#pragma unroll
    for (int v = 0; v < V; ++v) B[v] = JOINED && (cut >> k & 1) ? b[v] : fmaf(a[AV == 1 ? 0 : v], B[v], b[v]);
#pragma unroll
    for (int v = 0; v < AV; ++v) A[v] *= a[v];
  }
  if (!WIDE) wave_join<V, AV, false>(p, A, B, closed, eA, eB, eclosed);
  if (rl == RL - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sA[wave * p.W + cl * V + v] = A[AV == 1 ? 0 : v];
      sB[wave * p.W + cl * V + v] = B[v];
    }
    if (cl == 0) s_closed[wave] = closed;
  }
  if (threadIdx.x == 0) s_opened = cut & 1;
  __syncthreads();
  join_waves<V, SHARED, false>(p, q, slab, nw, sA, sB, s_closed, s_opened, carry);
  __syncthreads();
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float s = sB[wave * p.W + cl * V + v];
    h[v] = WIDE ? s : eclosed ? eB[v] : fmaf(eA[AV == 1 ? 0 : v], s, eB[v]);
  }
  const Turn<XT, V> ty(p.D, RL);
  int ends[K];
  const bool some = !WIDE && final && __any(last);
  if (some) segs_of<WIDE>(p, r, last, ends);
  cut = again<WIDE>(cut);
  first = again<WIDE>(first);
  if (!WHOLE) {
#pragma unroll
    for (int k = 0; k < K; ++k) x[k].again(), g[k].again();
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const ll at = r.p0 + k * r.step;
    if (!JOINED) cut_at<V, WIDE>(p, k, cut, first, h0, at, l.c, h);
    float a[AV], b[V];
    terms(k, a, b);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = JOINED && (cut >> k & 1) ? b[v] : fmaf(a[AV == 1 ? 0 : v], h[v], b[v]);
    if (l.ok) {
      if (turned) ty.put(buf, p.D, block, l.c, p.reverse, k, round_v<XT, V>(h));
      else if (full || (r.valid >> k & 1) || (p.zero_rest && (r.in >> k & 1))) store_v<XT, V>((y + at * p.D) + l.c, h);
      if (WIDE) {
        if (final && (last >> k & 1)) put_state<V>(p, final, at, l.c, h);
      } else if (some && ends[k] >= 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) final[(ll)ends[k] * p.D + l.c + v] = h[v];
      }
    }
  }
  if (turned) ty.store(buf, y + w0 * p.D);
}

template <typename XT, typename GT, int V, bool SHARED, bool WIDE>
void launch_fwd(const Launch& L, void* y, float* final, float* carry) {
  scan_fwd_kernel<XT, GT, V, SHARED, WIDE><<<L.blocks, L.g.nw * 64, L.lds, L.stream>>>(L.a, static_cast<XT*>(y), final, carry);
}

}  // namespace

extern "C" int tf_gated_scan_fwd(const TfGatedScan* d, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
                                 const float* h0, void* y, float* final, float* carry, float* workspace, size_t workspace_floats, tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_scan_fwd")) return rc;
  TF_REQUIRE(offsets && (d->n_rows == 0 || (gate && x && y && starts)), TF_EINVAL, "tf_gated_scan_fwd: null pointer");
  TF_REQUIRE(d->n_rows == 0 || index || (!h0 && !final), TF_EINVAL, "tf_gated_scan_fwd: h0 and final need an index");
  const size_t need = tf_gated_scan_workspace_floats(d, 0);
  TF_REQUIRE(workspace_floats >= need && (!need || (workspace && ((size_t)workspace & 7) == 0)), TF_ESHAPE,
             "tf_gated_scan_fwd: workspace too small, or not aligned to 8 bytes");
  Launch L;
  const void* like_x[2] = {y, nullptr};
  if (int rc = prepare(*d, "tf_gated_scan_fwd", gate, x, offsets, index, starts, h0, final != nullptr, workspace, stream, like_x, nullptr, 2, &L)) return rc;
  if (L.blocks) {
#define CALL(XT, GT, V, SH, WIDE) launch_fwd<XT, GT, V, SH, WIDE>(L, y, final, carry)
    TF_SCAN_DISPATCH(CALL, *d)
#undef CALL
  }
  TF_LAUNCH_CHECK("tf_gated_scan_fwd");
  return TF_OK;
}
