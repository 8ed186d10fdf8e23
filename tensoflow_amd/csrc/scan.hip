// Gated linear recurrence: geometry and sizes shared by both directions (scan_tile.h), and the one-token form.
#include "scan_tile.h"

namespace tfscan {

constexpr int TICKETS = 64;  // 256 bytes from counter to counter

static int pow2_from(int n) {
  int p = 1;
  while (p < n) p <<= 1;
  return p;
}

// Depends on sizes alone (not on addresses or strides): the backward pass cuts the tiles that the forward pass cut.
Geo geometry(const TfGatedScan& d) {
  Geo g = {};
  const int D = d.channels, G = d.gates, P = D / G;
  g.shared = P > 1;
  const int unit = g.shared ? P : D;  // what a lane's channels have to divide
  g.V = unit % 4 == 0 ? 4 : unit % 3 == 0 ? 3 : unit % 2 == 0 ? 2 : 1;
  const int lanes = unit / g.V;
  if (!g.shared) {
    g.CL = lanes < 64 ? pow2_from(lanes) : 64;
    g.LP = g.hs = g.parts = 1;
    g.slabs = (lanes + 63) / 64;
  } else if (lanes <= 64) {
    g.LP = lanes;
    g.hs = 64 / lanes < G ? 64 / lanes : G;
    g.CL = pow2_from(g.hs * lanes);
    g.parts = 1;
    g.slabs = (G + g.hs - 1) / g.hs;
  } else {
    g.LP = g.CL = 64;
    g.hs = 1;
    g.parts = (lanes + 63) / 64;
    g.slabs = G * g.parts;
  }
  g.W = g.CL * g.V;
  const ll wave_rows = (64 / g.CL) * K;
  // waves of a workgroup: as many as leave two workgroups to every CU, or as hold all rows in one tile
  // (four at most where rows are shorter than a cache line: their buffers take 9 KB of LDS a wave; and for fp32, most of whose kernels' registers leave
  // room for 12 waves on a CU: three workgroups of four, where eight waves would be alone)
  const int most = d.x_type == TF_TYPE_F32 || D < 64 ? 4 : 8;
  g.nw = most;
  while (g.nw > 1 && ((d.n_rows + g.nw * wave_rows - 1) / (g.nw * wave_rows)) * g.slabs < 512) g.nw >>= 1;
  int all = 1;  // waves that hold all rows, no more than that
  while (all < most && d.n_rows > all * wave_rows) all <<= 1;
  if (d.n_rows <= all * wave_rows) g.nw = all;
  g.tile_rows = g.nw * wave_rows;
  g.tiles = (d.n_rows + g.tile_rows - 1) / g.tile_rows;
  return g;
}

int check_desc(const TfGatedScan* d, const char* who) {
  TF_REQUIRE(d, TF_EINVAL, "%s: null descriptor", who);
  TF_REQUIRE(d->n_rows >= 0 && d->n_segments >= 0, TF_ESHAPE, "%s: negative size", who);
  TF_REQUIRE(d->channels >= 1 && d->channels <= 65536 && d->gates >= 1 && d->channels % d->gates == 0, TF_ESHAPE,
             "%s: channels must be 1..65536 and a multiple of the gates", who);
  TF_REQUIRE(d->n_rows < (1ll << 38) && d->n_segments < (1ll << 31), TF_ESHAPE, "%s: too many rows or segments", who);
  TF_REQUIRE(d->n_rows <= 1 || (d->ld_x >= 0 && d->ld_gate >= 0), TF_ESHAPE, "%s: negative row stride", who);
  TF_REQUIRE((d->x_type == TF_TYPE_F32 || d->x_type == TF_TYPE_F16 || d->x_type == TF_TYPE_BF16) && (d->gate_type == d->x_type || d->gate_type == TF_TYPE_F32), TF_EINVAL,
             "%s: types must be fp32, fp16 or bf16, and the gate's that of x or fp32", who);
  TF_REQUIRE(d->form == TF_GATE_DECAY || d->form == TF_GATE_LOG || d->form == TF_GATE_ALPHA, TF_EINVAL, "%s: unknown gate form", who);
  return TF_OK;
}


// floats of the words, the ends and the counter that tiles wait for each other with (none for a single tile)
static size_t groups_of(const Geo& g) { return g.tiles / GRP; }
size_t chain_floats(const TfGatedScan& d, const Geo& g) {
  if (g.tiles <= 1) return 0;
  const size_t ends = groups_of(g) / GRP * d.channels;
  return 2 * ((size_t)g.tiles + groups_of(g)) * d.channels + (ends + 1) / 2 * 2 + (size_t)g.slabs * TICKETS;
}
size_t parts_floats(const TfGatedScan& d, const Geo& g) { return g.shared && g.parts > 1 ? (size_t)g.parts * d.n_rows * d.gates : 0; }

static bool fits(const void* p, size_t bytes) { return ((size_t)p & (bytes - 1)) == 0; }

static __global__ void __launch_bounds__(256) scan_clear_kernel(ull* __restrict__ words, ll n, ll all) {
  const ll i = (ll)blockIdx.x * 256 + threadIdx.x;
  if (i < all) words[i] = i < n ? EMPTY : 0;
}

// Arguments, chain memory cleared, grid.  like_x: two further arrays laid out as a contiguous x, like_gate: one as a contiguous gate (each may be null);
// lds_floats: for each wave and channel.
int prepare(const TfGatedScan& d, const char* who, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
            const float* h0, bool empties, float* workspace, tf_stream_t stream, const void* const* like_x, const void* like_gate, int lds_floats, Launch* out) {
  const Geo g = geometry(d);
  const size_t xs = d.x_type == TF_TYPE_F32 ? 4 : 2, gs = d.gate_type == TF_TYPE_F32 ? 4 : 2;
  const int vx = g.V == 3 ? 1 : g.V, vg = g.shared ? 1 : vx;
  ScanArgs a = {};
  a.gate = gate;
  a.x = x;
  a.offsets = (const ll*)offsets;
  a.index = (const ll*)index;
  a.starts = (const ull*)starts;
  a.h0 = h0;
  a.n_rows = d.n_rows;
  a.n_seg = d.n_segments;
  a.ld_x = d.ld_x;
  a.ld_gate = d.ld_gate;
  a.D = d.channels;
  a.G = d.gates;
  a.P = d.channels / d.gates;
  a.form = d.form;
  a.reverse = d.reverse != 0;
  a.zero_rest = d.zero_rest != 0;
  a.CL = g.CL;
  a.W = g.W;
  a.LP = g.LP;
  a.hs = g.hs;
  a.parts = g.parts;
  a.slabs = g.slabs;
  auto all = [&](size_t bx, size_t bg) {
    return fits(x, bx) && fits(like_x[0], bx) && fits(like_x[1], bx) && fits(gate, bg) && fits(like_gate, bg);
  };
  TF_REQUIRE(all(vx * xs, vg * gs) && (d.n_rows <= 1 || (d.ld_x % vx == 0 && d.ld_gate % vg == 0)), TF_EINVAL,
             "%s: rows of x must be aligned to %d elements, of the gate to %d", who, vx, vg);
  const size_t join = ((size_t)g.nw * g.W * lds_floats + 3) / 4 * 16;
  // rows shorter than a cache line, side by side in memory: turned in LDS
  if (g.slabs == 1 && d.channels * xs < 128 && all(16, 16) && d.ld_x == d.channels && d.ld_gate == d.gates) {
    const size_t row = d.channels * xs > d.gates * gs ? d.channels * xs : d.gates * gs;
    a.narrow = (int)(64 / g.CL * (K * row + 16));
  }
  const ll rest = empties ? (d.n_segments + 64ll * g.nw - 1) / (64ll * g.nw) : 0, blocks = g.tiles * g.slabs + rest;
  TF_REQUIRE(blocks < (1ll << 31) - 1, TF_ESHAPE, "%s: too many rows", who);
  a.tiles = (int)g.tiles;
  hipStream_t st = (hipStream_t)stream;
  if (g.tiles > 1) {
    a.words = reinterpret_cast<ull*>(workspace);
    a.groups = a.words + g.tiles * d.channels;
    a.ends = reinterpret_cast<unsigned*>(a.groups + groups_of(g) * d.channels);
    const ll all = (ll)(chain_floats(d, g) / 2), n = all - (ll)g.slabs * TICKETS / 2;
    a.ticket = reinterpret_cast<unsigned*>(a.words + n);
    a.tickets = TICKETS;
    scan_clear_kernel<<<(unsigned)((all + 255) / 256), 256, 0, st>>>(a.words, n, all);
  }
  *out = {a, g, (unsigned)blocks, join + (size_t)g.nw * a.narrow, st};
  return TF_OK;
}

}  // namespace tfscan

using namespace tfscan;

namespace {

// A workgroup is a row and 256 V of its channels.  Bound: the launch for a few rows (one of 2048 channels 2.3 us), then the states, read and written
// (256 x 4096 bf16 with 32 fp32 gates: 4.8 us, 2.6 TB/s).  The first row of a slot takes the later ones of the same slot along, in order; the others leave.
template <typename XT, typename GT, int V, bool SHARED>
__global__ void __launch_bounds__(256) step_kernel(TfGatedScan d, const GT* __restrict__ gate, const XT* __restrict__ x, const ll* __restrict__ slots,
                                                   ll n_slots, float* __restrict__ state, XT* __restrict__ y) {
  constexpr int AV = SHARED ? 1 : V;
  const int D = d.channels, P = D / d.gates, n = (int)d.n_rows, r = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * V;
  const bool mine = c < D;
  const ll slot = slots[r];
  if (slot < 0 || slot >= n_slots) {
    const float z[V] = {};
    if (d.zero_rest && mine) store_v<XT, V>(y + (ll)r * D + c, z);
    return;
  }
  const ll g = SHARED ? c / P : c;
  Raw<XT, V> rx;
  Raw<GT, AV> rg;
  float h[V];
  if (mine) {  // asked for before the search, which needs none of it
    rx = load_v<XT, V>(x + r * d.ld_x + c);
    rg = load_v<GT, AV>(gate + r * d.ld_gate + g);
    const Raw<float, V> s = load_v<float, V>(state + slot * D + c);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = s[v];
  }
  int last = r;
  if (n > 1) {
    int before = 0, behind = 0;
    for (int q = threadIdx.x; q < n; q += 256) {
      const bool same = slots[q] == slot;
      before |= same && q < r;
      behind |= same && q > r;
    }
    if (__syncthreads_or(before)) return;
    if (__syncthreads_or(behind)) last = n - 1;
  }
  if (!mine) return;
  for (int q = r; q <= last; ++q) {
    if (q != r) {
      if (slots[q] != slot) continue;
      rx = load_v<XT, V>(x + q * d.ld_x + c);
      rg = load_v<GT, AV>(gate + q * d.ld_gate + g);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = rg[AV == 1 ? 0 : v], b = rx[v];
      if (d.form == TF_GATE_LOG) a = exp_gate(a);
      if (d.form == TF_GATE_ALPHA) b *= a, a = 1.f - a;
      h[v] = fmaf(a, h[v], b);
    }
    store_v<XT, V>(y + (ll)q * D + c, h);
  }
  store_v<float, V>(state + slot * D + c, h);
}

}  // namespace

extern "C" size_t tf_gated_scan_carry_floats(const TfGatedScan* d) {
  if (!d || check_desc(d, "tf_gated_scan_carry_floats")) return 0;
  return (size_t)geometry(*d).tiles * d->channels;
}
extern "C" size_t tf_gated_scan_workspace_floats(const TfGatedScan* d, int32_t backward) {
  if (!d || check_desc(d, "tf_gated_scan_workspace_floats")) return 0;
  const Geo g = geometry(*d);
  return chain_floats(*d, g) + (backward ? parts_floats(*d, g) : 0);
}

extern "C" int tf_gated_step(const TfGatedScan* d, const void* gate, const void* x, const int64_t* slots, int64_t n_slots, float* state, void* y,
                             tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_step")) return rc;
  TF_REQUIRE(n_slots >= 0 && d->n_rows <= 8192, TF_ESHAPE, "tf_gated_step: a negative pool size, or over 8192 rows");
  if (d->n_rows == 0) return TF_OK;
  TF_REQUIRE(gate && x && slots && y && (n_slots == 0 || state), TF_EINVAL, "tf_gated_step: null pointer");
  // four channels a lane, unless that leaves most of the card idle: one row of 2048 channels is 8 workgroups at one channel a lane
  const bool shared = d->channels != d->gates;
  const int unit = shared ? d->channels / d->gates : d->channels;
  const size_t xs = d->x_type == TF_TYPE_F32 ? 4 : 2, gs = d->gate_type == TF_TYPE_F32 ? 4 : 2;
  const int vg = shared ? 1 : 4;
  const bool aligned = fits(x, 4 * xs) && fits(y, 4 * xs) && fits(gate, vg * gs) && fits(state, 16) && (d->n_rows == 1 || (d->ld_x % 4 == 0 && d->ld_gate % vg == 0));
  const int V = unit % 4 == 0 && aligned && d->n_rows * d->channels >= 65536 ? 4 : 1;
  const dim3 grid((unsigned)((d->channels + 256 * V - 1) / (256 * V)), (unsigned)d->n_rows);
  hipStream_t st = (hipStream_t)stream;
#define STEP(XT, GT, VV, SH) step_kernel<XT, GT, VV, SH><<<grid, 256, 0, st>>>(*d, static_cast<const GT*>(gate), static_cast<const XT*>(x), (const ll*)slots, n_slots, state, static_cast<XT*>(y))
#define STEP_V(XT, GT)                                                            \
  if (V == 4) { if (shared) STEP(XT, GT, 4, true); else STEP(XT, GT, 4, false); } \
  else { if (shared) STEP(XT, GT, 1, true); else STEP(XT, GT, 1, false); }
  if (d->x_type == TF_TYPE_F32) { STEP_V(float, float) }
  else if (d->x_type == TF_TYPE_F16 && d->gate_type == TF_TYPE_F16) { STEP_V(f16, f16) }
  else if (d->x_type == TF_TYPE_F16) { STEP_V(f16, float) }
  else if (d->gate_type == TF_TYPE_BF16) { STEP_V(bf16, bf16) }
  else { STEP_V(bf16, float) }
#undef STEP_V
#undef STEP
  TF_LAUNCH_CHECK("tf_gated_step");
  return TF_OK;
}
