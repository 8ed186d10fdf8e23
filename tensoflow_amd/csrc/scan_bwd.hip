// Gradients of the gated linear recurrence over a packed batch (scan_tile.h has the decomposition).  l_t, the gradient of h_t:
//   l_t = gy_t + m_{t+1}, m_t = a_t l_t (a segment's last row takes gfinal for m_{t+1}); d b_t = l_t; d a_t = l_t h_{t-1}; d h0 = m_0.
//   TF_GATE_DECAY: dx = l, dg = l h_{t-1};   TF_GATE_LOG: dx = l, dg = l a h_{t-1};   TF_GATE_ALPHA: dx = g l, dg = l (x - h_{t-1}).
// The states are computed again, in fp32, from the state in front of the tile that the forward pass kept: x is read where y would be, and no rounding of
// y enters.  m runs over the tiles as h does, from the last to the first: what the tile hands to the tile before it is A m + B with A = prod a.
#include "scan_tile.h"

using namespace tfscan;

namespace {

// sums over the LP lanes of a head of K values: the first lane has them all
template <int K>
__device__ __forceinline__ void head_sums(float (&s)[K], int wl, int LP) {
  for (int o = 1; o < LP; o <<= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const float z = __shfl_down(s[k], o);
      if (wl + o < LP) s[k] += z;
    }
  }
}
// LP = 2^n >= K: halves of the values change sides, so that K - 1 shuffles do what K for each doubling did, and one for each further doubling; lane wl has the
// sum of the row that has wl's low bits in reversed order
template <int K>
__device__ __forceinline__ float head_sums_pow2(float (&s)[K], int wl, int LP) {
#pragma unroll
  for (int n = K / 2, o = 1; n >= 1; n >>= 1, o <<= 1) {
    const bool up = wl & o;
#pragma unroll
    for (int k = 0; k < K / 2; ++k) {
      if (k >= n) break;
      const float give = up ? s[k] : s[k + n], keep = up ? s[k + n] : s[k];
      s[k] = keep + __shfl_xor(give, o);
    }
  }
  float v = s[0];
  for (int o = K; o < LP; o <<= 1) v += __shfl_xor(v, o);
  return v;
}

// Registers: 16-bit values stay packed.  With shared gates and a wave across the channels that takes 98 to 115 vector registers, two workgroups of eight waves
// on a CU (16385 x 2048 bf16 with 16 gates: 81 us, 119 with x and gy widened and one workgroup).  The other kernels of four 16-bit channels take 135 to
// 172: one workgroup of eight waves, or two to three of four (rows under 64 channels).  fp32 takes 94 to 167, three workgroups of four waves or more; its
// narrow kernels of three and four channels a lane 176 to 230, two of them.  The bound of 2 waves squeezes none of them and has to stay so:
// held to 128 registers, a kernel of 4 x 16-bit channels spilled 63 and one of its four channels came out with wrong states.  No mistake was found in
// the source (run on the CPU, a thread for each lane, it is right and clean under the address, undefined-behaviour, memory and thread sanitizers), so
// no_spills.py ends the build of such a kernel.  Scalar registers are spilled in all of them, 102 to 181, into lanes of vector registers.
// Measured: 40001 x 512 fp32, a gate for each channel, 102 us (491 MB of which 328 here: 4.1 TB/s of its own reads and writes).
template <typename XT, typename GT, int V, bool SHARED, bool WIDE>
__global__ void __launch_bounds__(512, 2) scan_bwd_kernel(ScanArgs p, const float* __restrict__ carry, const XT* __restrict__ gy, const float* __restrict__ gfinal,
                                                       GT* __restrict__ dgate, float* __restrict__ dgate_parts, XT* __restrict__ dx, float* __restrict__ dh0) {
  extern __shared__ __attribute__((aligned(16))) float smem[];
  __shared__ unsigned s_ticket;
  __shared__ int s_closed[8], s_mclosed[8], s_opened;
  constexpr int AV = SHARED ? 1 : V;
  const int nw = blockDim.x >> 6, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  float *sA = smem, *sB = sA + nw * p.W, *sP = sB + nw * p.W, *sQ = sP + nw * p.W;
  char* buf = reinterpret_cast<char*>(smem + (4 * nw * p.W + 3 & ~3)) + wave * p.narrow;
  const ll lo = max(p.offsets[0], 0ll), hi = min(p.offsets[p.n_seg], p.n_rows);
  int slab;
  const int qd = take_job(p, &s_ticket, slab), q = p.tiles - 1 - qd;  // the tiles from the last to the first
  if (slab < 0) {
    empty_segments(p, (ll)qd * nw + wave, gfinal, dh0);
    return;
  }
  const int cl = WIDE ? lane : lane & (p.CL - 1), rl = WIDE ? 0 : lane / p.CL, RL = WIDE ? 1 : 64 / p.CL, T = nw * RL * K;
  const Lane<V, SHARED> l(p, slab, cl);
  const Rows<WIDE> r(p, (ll)q * T + (wave * RL + rl) * K, T, lo, hi);
  const ll t0 = (ll)(p.reverse ? p.tiles - 1 - q : q) * T;
  const ll w0 = t0 + (ll)(p.reverse ? nw - 1 - wave : wave) * RL * K;
  const int block = p.reverse ? RL - 1 - rl : rl;
  const bool full = t0 >= lo && t0 + T <= hi, turned = !WIDE && p.narrow && full;
  Raw<XT, V> x[K], ry[K];
  Raw<GT, AV> g[K];
  unsigned first, last;
  if (turned) {
    Turn<XT, V> tx(p.D, RL), ty(p.D, RL);
    Turn<GT, AV> tg(p.G, RL);
    tx.load(static_cast<const XT*>(p.x) + w0 * p.D);
    tg.load(static_cast<const GT*>(p.gate) + w0 * p.G);
    if (gy) ty.load(gy + w0 * p.D);
    r.bits(p, hi, first, last);
    tx.to_rows(buf, p.D, block, l.c, p.reverse, x);
    tg.to_rows(buf, p.G, block, l.g, p.reverse, g);
    if (gy) ty.to_rows(buf, p.D, block, l.c, p.reverse, ry);
  } else {
    direct_rows<XT, V, WIDE>(static_cast<const XT*>(p.x), p.ld_x, r, l.c, full, x);
    direct_rows<GT, AV, WIDE>(static_cast<const GT*>(p.gate), p.ld_gate, r, l.g, full, g);
    if (gy) direct_rows<XT, V, WIDE>(gy, p.D, r, l.c, full, ry);
    r.bits(p, hi, first, last);
  }
  if (!gy) {
#pragma unroll
    for (int k = 0; k < K; ++k) ry[k].zero();
  }
#pragma unroll
  for (int k = 0; k < K; ++k) gates_kept<GT, AV>(g[k], p.form);
  bool alpha = p.form == TF_GATE_ALPHA;
  const bool logs = p.form == TF_GATE_LOG;
  const float s1 = alpha ? -1.f : 1.f, s0 = alpha ? 1.f : 0.f;
  const unsigned none = ~r.valid & ((1u << K) - 1);
  unsigned cut = first | none, mcut = last | none;
  // for all of a lane's rows at once: what comes from behind a segment's end, added to gy where that is fp32; the states that segments begin from
  const float *h0 = p.h0, *gf = gfinal;
  constexpr bool WHOLE = sizeof(XT) == 4;
  int seg0[K];
  float begin[K][V];
  if (!WIDE && WHOLE && gf) {
    if (__any(last)) {
      int seg[K];
      float s[K][V];
      segs_of<WIDE>(p, r, last, seg);
      states_of<V>(p, gf, seg, l.c, s);
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) ry[k].w[v] = __builtin_bit_cast(unsigned, seg[k] >= 0 ? ry[k][v] + s[k][v] : ry[k][v]);
    }
    gf = nullptr;
  }
  const bool some = !WIDE && (p.h0 || dh0) && __any(first);
  if (some) segs_of<WIDE>(p, r, first, seg0);
  const bool began = !WIDE && WHOLE && h0 && some;
  if (began) states_of<V>(p, h0, seg0, l.c, begin);
  if (!WIDE && WHOLE) h0 = nullptr;
  float A[AV], B[V], eA[AV], eB[V], P[AV], Q[V], eP[AV], eQ[V];
  bool closed = cut != 0, eclosed, mclosed = mcut != 0, emclosed;
#pragma unroll
  for (int v = 0; v < AV; ++v) A[v] = 1.f;
#pragma unroll
  for (int v = 0; v < V; ++v) B[v] = Q[v] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    cut_at<V, WIDE>(p, k, cut, first, h0, r.p0 + k * r.step, l.c, B);
    if (!WIDE && WHOLE && began) {
#pragma unroll
      for (int v = 0; v < V; ++v) B[v] = seg0[k] >= 0 ? begin[k][v] : B[v];
    }
    float ga[AV];
    gates_of<GT, AV>(g[k], p.form, ga);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float gav = ga[AV == 1 ? 0 : v];
      B[v] = fmaf(fmaf(gav, s1, s0), B[v], alpha ? gav * x[k][v] : x[k][v]);
    }
#pragma unroll
    for (int v = 0; v < AV; ++v) A[v] *= fmaf(ga[v], s1, s0);
  }
#pragma unroll
  for (int v = 0; v < AV; ++v) P[v] = A[v];
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    cut_at<V, WIDE>(p, k, mcut, last, gf, r.p0 + k * r.step, l.c, Q);
    float ga[AV];
    gates_of<GT, AV>(g[k], p.form, ga);
#pragma unroll
    for (int v = 0; v < V; ++v) Q[v] = fmaf(ga[AV == 1 ? 0 : v], s1, s0) * (ry[k][v] + Q[v]);
  }
  if (!WIDE) {
    wave_join<V, AV, false>(p, A, B, closed, eA, eB, eclosed);
    wave_join<V, AV, true>(p, P, Q, mclosed, eP, eQ, emclosed);
  }
  if (rl == RL - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sA[wave * p.W + cl * V + v] = A[AV == 1 ? 0 : v];
      sB[wave * p.W + cl * V + v] = B[v];
    }
    if (cl == 0) s_closed[wave] = closed;
  }
  if (rl == 0) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sP[wave * p.W + cl * V + v] = P[AV == 1 ? 0 : v];
      sQ[wave * p.W + cl * V + v] = Q[v];
    }
    if (cl == 0) s_mclosed[wave] = mclosed;
  }
  if (threadIdx.x == blockDim.x - 1) s_opened = mcut >> (K - 1) & 1;
  __syncthreads();
  for (int i = threadIdx.x; i < p.W; i += nw * 64) {
    const Lane<V, SHARED> ln(p, slab, i / V);
    if (!ln.ok) continue;
    float h = carry[(ll)q * p.D + ln.c + i % V];
    for (int w = 0; w < nw; ++w) {
      const float b = sB[w * p.W + i];
      sB[w * p.W + i] = h;
      h = s_closed[w] ? b : fmaf(sA[w * p.W + i], h, b);
    }
  }
  join_waves<V, SHARED, true>(p, qd, slab, nw, sP, sQ, s_mclosed, s_opened, nullptr);
  __syncthreads();
  float h[V], m[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float s = sB[wave * p.W + cl * V + v], z = sQ[wave * p.W + cl * V + v];
    h[v] = WIDE ? s : eclosed ? eB[v] : fmaf(eA[AV == 1 ? 0 : v], s, eB[v]);
    m[v] = WIDE ? z : emclosed ? eQ[v] : fmaf(eP[AV == 1 ? 0 : v], z, eQ[v]);
  }
  cut = again<WIDE>(cut);
  mcut = again<WIDE>(mcut);
  first = again<WIDE>(first);
  last = again<WIDE>(last);
#pragma unroll
  for (int k = 0; k < K; ++k) x[k].again(), g[k].again(), ry[k].again();
  // from the last row to the first: l takes the place of gy, x and the gates stay
  float lam[K][V];
  const Turn<XT, V> tx(p.D, RL);
  const Turn<GT, AV> tg(p.G, RL);
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    const ll at = r.p0 + k * r.step;
    float o[V];
    cut_at<V, WIDE>(p, k, mcut, last, gf, at, l.c, m);
    float ga[AV];
    gates_of<GT, AV>(g[k], p.form, ga);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float gav = ga[AV == 1 ? 0 : v], z = ry[k][v] + m[v];
      lam[k][v] = z;
      o[v] = alpha ? gav * z : z;
      m[v] = fmaf(gav, s1, s0) * z;
    }
    if (dx && l.ok) {
      if (turned) tx.put(buf, p.D, block, l.c, p.reverse, k, round_v<XT, V>(o));
      else if (full || (r.valid >> k & 1) || (p.zero_rest && (r.in >> k & 1))) store_v<XT, V>((dx + at * p.D) + l.c, o);
    }
    if (WIDE) {
      if (dh0 && l.ok && (first >> k & 1)) put_state<V>(p, dh0, at, l.c, m);
    } else if (dh0 && some && l.ok && seg0[k] >= 0) {
#pragma unroll
      for (int v = 0; v < V; ++v) dh0[(ll)seg0[k] * p.D + l.c + v] = m[v];
    }
  }
  if (turned && dx) tx.store(buf, dx + w0 * p.D);
  if (!dgate) return;
  if (began) states_of<V>(p, p.h0, seg0, l.c, begin);
  // from the first row to the last: the states in front of the rows, and the gate's gradient
  float sums[K];
  Raw<GT, AV> og[K];
#pragma unroll
  for (int k = 0; k < K; ++k) x[k].again(), g[k].again();
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const ll at = r.p0 + k * r.step;
    float d[V], ga[AV];
    gates_of<GT, AV>(g[k], p.form, ga);
    cut_at<V, WIDE>(p, k, cut, first, h0, at, l.c, h);
    if (!WIDE && WHOLE && began) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = seg0[k] >= 0 ? begin[k][v] : h[v];
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float gav = ga[AV == 1 ? 0 : v];
      d[v] = lam[k][v] * (alpha ? x[k][v] - h[v] : logs ? gav * h[v] : h[v]);
      h[v] = fmaf(fmaf(gav, s1, s0), h[v], alpha ? gav * x[k][v] : x[k][v]);
    }
    if (!SHARED) {
      og[k] = round_v<GT, AV>(d);
      if (!turned && l.ok && (full || (r.valid >> k & 1) || (p.zero_rest && (r.in >> k & 1)))) store_v<GT, AV>(dgate + at * p.G + l.g, d);
    } else {
      sums[k] = 0.f;
#pragma unroll
      for (int v = 0; v < V; ++v) sums[k] += d[v];
      if (!l.ok) sums[k] = 0.f;
    }
  }
  if (SHARED) {
    if (p.LP >= K && (p.LP & (p.LP - 1)) == 0 && !turned) {
      const float s = head_sums_pow2<K>(sums, l.wl, p.LP);
      const int k = __brev(l.wl) >> (33 - __ffs(K));
      const ll at = r.p0 + k * r.step;
      if (l.wl < K && l.head && ((r.valid >> k & 1) || (p.zero_rest && (r.in >> k & 1)))) {
        if (dgate_parts) dgate_parts[((ll)l.part * p.n_rows + at) * p.G + l.g] = s;
        else dgate[at * p.G + l.g] = from_f<GT>(s);
      }
      return;
    }
    head_sums<K>(sums, l.wl, p.LP);
    if (!turned) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const ll at = r.p0 + k * r.step;
        if (l.ok && l.wl == 0 && ((r.valid >> k & 1) || (p.zero_rest && (r.in >> k & 1)))) {
          if (dgate_parts) dgate_parts[((ll)l.part * p.n_rows + at) * p.G + l.g] = sums[k];
          else dgate[at * p.G + l.g] = from_f<GT>(sums[k]);
        }
      }
      return;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) og[k] = round_v<GT, AV>(&sums[k]);
  }
  if (turned) {
    wave_fence();
    if (l.ok && l.wl == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) tg.put(buf, p.G, block, l.g, p.reverse, k, og[k]);
    }
    tg.store(buf, dgate + w0 * p.G);
  }
}

// heads wider than a workgroup's channels: the gate's gradient from its pieces, in their order
template <typename GT>
__global__ void __launch_bounds__(256) scan_gate_parts_kernel(const float* __restrict__ in, const ll* __restrict__ offsets, ll n_seg, ll n_rows, int G, int parts,
                                                              int zero_rest, GT* __restrict__ dgate) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x, i = e / G;
  if (i >= n_rows || (!zero_rest && (i < offsets[0] || i >= offsets[n_seg]))) return;
  float s = 0.f;
  for (int k = 0; k < parts; ++k) s += in[k * n_rows * G + e];
  dgate[e] = from_f<GT>(s);
}

struct BwdPtrs {
  const float* carry;
  const void* gy;
  const float* gfinal;
  void* dgate;
  float* parts;
  void* dx;
  float* dh0;
};
template <typename XT, typename GT, int V, bool SHARED, bool WIDE>
void launch_bwd(const Launch& L, const BwdPtrs& b) {
  scan_bwd_kernel<XT, GT, V, SHARED, WIDE><<<L.blocks, L.g.nw * 64, L.lds, L.stream>>>(L.a, b.carry, static_cast<const XT*>(b.gy), b.gfinal, static_cast<GT*>(b.dgate),
                                                                                 b.parts, static_cast<XT*>(b.dx), b.dh0);
}

}  // namespace

extern "C" int tf_gated_scan_bwd(const TfGatedScan* d, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
                                 const float* h0, const float* carry, const void* gy, const float* gfinal, void* dgate, void* dx, float* dh0, float* workspace,
                                 size_t workspace_floats, tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_scan_bwd")) return rc;
  TF_REQUIRE(offsets && (d->n_rows == 0 || (gate && x && starts && carry)), TF_EINVAL, "tf_gated_scan_bwd: null pointer");
  TF_REQUIRE(d->n_rows == 0 || index || (!h0 && !gfinal && !dh0), TF_EINVAL, "tf_gated_scan_bwd: h0 and final need an index");
  const size_t need = tf_gated_scan_workspace_floats(d, 1);
  TF_REQUIRE(workspace_floats >= need && (!need || (workspace && ((size_t)workspace & 7) == 0)), TF_ESHAPE,
             "tf_gated_scan_bwd: workspace too small, or not aligned to 8 bytes");
  Launch L;
  const Geo g = geometry(*d);
  const void* like_x[2] = {gy, dx};
  if (int rc = prepare(*d, "tf_gated_scan_bwd", gate, x, offsets, index, starts, h0, dh0 != nullptr, workspace, stream, like_x, dgate, 4, &L)) return rc;
  const BwdPtrs b = {carry, gy, gfinal, dgate, parts_floats(*d, g) ? workspace + chain_floats(*d, g) : nullptr, dx, dh0};
  const ll pblocks = b.parts && dgate ? (d->n_rows * (ll)d->gates + 255) / 256 : 0;
  TF_REQUIRE(pblocks < (1ll << 31), TF_ESHAPE, "tf_gated_scan_bwd: too many rows");
  if (L.blocks) {
#define CALL(XT, GT, V, SH, WIDE) launch_bwd<XT, GT, V, SH, WIDE>(L, b)
    TF_SCAN_DISPATCH(CALL, *d)
#undef CALL
  }
  if (pblocks) {
    hipStream_t st = (hipStream_t)stream;
#define PARTS(GT) scan_gate_parts_kernel<GT><<<(unsigned)pblocks, 256, 0, st>>>(b.parts, (const ll*)offsets, d->n_segments, d->n_rows, d->gates, g.parts, d->zero_rest, static_cast<GT*>(dgate))
    if (d->gate_type == TF_TYPE_F32) PARTS(float);
    else if (d->gate_type == TF_TYPE_F16) PARTS(f16);
    else PARTS(bf16);
#undef PARTS
  }
  TF_LAUNCH_CHECK("tf_gated_scan_bwd");
  return TF_OK;
}
