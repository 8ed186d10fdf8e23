// Gated linear recurrence over a packed batch of sequences, h_t = a_t h_{t-1} + b_t, its gradients and its one-token form.
//   TF_GATE_DECAY: a = g, b = x;   TF_GATE_LOG: a = exp(g), b = x;   TF_GATE_ALPHA: a = 1 - g, b = g x (compositing).
// Backward, l_t the gradient of h_t: l_t = gy_t + a_{t+1} l_{t+1}; d b_t = l_t; d a_t = l_t h_{t-1}; d h0 = a_0 l_0.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "tf_common.h"

namespace {

typedef long long ll;

__device__ __forceinline__ float load1(const void* p, ll i, int type) {
  if (type == TF_TYPE_F32) return static_cast<const float*>(p)[i];
  if (type == TF_TYPE_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __hip_bfloat16*>(p)[i]);
}
// the one rounding of a result to its type: to nearest, ties to even
__device__ __forceinline__ void store1(void* p, ll i, int type, float v) {
  if (type == TF_TYPE_F32) static_cast<float*>(p)[i] = v;
  else if (type == TF_TYPE_F16) static_cast<__half*>(p)[i] = __float2half(v);
  else static_cast<__hip_bfloat16*>(p)[i] = __float2bfloat16(v);
}
__device__ __forceinline__ void gate_terms(int form, float g, float x, float& a, float& b) {
  a = form == TF_GATE_LOG ? expf(g) : form == TF_GATE_ALPHA ? 1.f - g : g;
  b = form == TF_GATE_ALPHA ? g * x : x;
}

struct Scan {
  TfGatedScan d;
  const void *gate, *x;
  const ll* offsets;
  const float* h0;
};

__device__ __forceinline__ void seg_range(const Scan& p, ll s, ll& lo, ll& hi) {
  lo = min(max(p.offsets[s], 0ll), (ll)p.d.n_rows);
  hi = min(max(p.offsets[s + 1], lo), (ll)p.d.n_rows);
}

// one thread per (segment, channel), row after row
__global__ void __launch_bounds__(256) scan_fwd_kernel(Scan p, void* __restrict__ y, float* __restrict__ final) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x;
  const int D = p.d.channels, P = D / p.d.gates;
  if (e >= p.d.n_segments * (ll)D) return;
  const ll s = e / D;
  const int c = (int)(e % D);
  ll lo, hi;
  seg_range(p, s, lo, hi);
  float h = p.h0 ? p.h0[e] : 0.f;
  for (ll k = lo; k < hi; ++k) {
    const ll i = p.d.reverse ? hi - 1 - (k - lo) : k;
    float a, b;
    gate_terms(p.d.form, load1(p.gate, i * p.d.ld_gate + c / P, p.d.gate_type), load1(p.x, i * p.d.ld_x + c, p.d.x_type), a, b);
    h = fmaf(a, h, b);
    store1(y, i * D + c, p.d.x_type, h);
  }
  if (final) final[e] = h;
}

// one thread per (segment, channel): the states again, row after row, then the gradients from the last row to the first;
// work [n_rows, channels] holds h_{t-1}, then the channel's share of the gate's gradient
__global__ void __launch_bounds__(256) scan_bwd_kernel(Scan p, const void* __restrict__ gy, const float* __restrict__ gfinal, float* __restrict__ work,
                                                       void* __restrict__ dx, float* __restrict__ dh0) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x;
  const int D = p.d.channels, P = D / p.d.gates;
  if (e >= p.d.n_segments * (ll)D) return;
  const ll s = e / D;
  const int c = (int)(e % D);
  ll lo, hi;
  seg_range(p, s, lo, hi);
  float h = p.h0 ? p.h0[e] : 0.f;
  for (ll k = lo; k < hi; ++k) {
    const ll i = p.d.reverse ? hi - 1 - (k - lo) : k;
    float a, b;
    gate_terms(p.d.form, load1(p.gate, i * p.d.ld_gate + c / P, p.d.gate_type), load1(p.x, i * p.d.ld_x + c, p.d.x_type), a, b);
    work[i * D + c] = h;
    h = fmaf(a, h, b);
  }
  float l = gfinal ? gfinal[e] : 0.f;
  for (ll k = hi - 1; k >= lo; --k) {
    const ll i = p.d.reverse ? hi - 1 - (k - lo) : k;
    const float g = load1(p.gate, i * p.d.ld_gate + c / P, p.d.gate_type), x = load1(p.x, i * p.d.ld_x + c, p.d.x_type);
    float a, b;
    gate_terms(p.d.form, g, x, a, b);
    if (gy) l += load1(gy, i * D + c, p.d.x_type);
    const float before = work[i * D + c];
    work[i * D + c] = p.d.form == TF_GATE_ALPHA ? l * (x - before) : p.d.form == TF_GATE_LOG ? l * before * a : l * before;
    if (dx) store1(dx, i * D + c, p.d.x_type, p.d.form == TF_GATE_ALPHA ? g * l : l);
    l *= a;
  }
  if (dh0) dh0[e] = l;
}

__global__ void __launch_bounds__(256) scan_gate_grad_kernel(Scan p, const float* __restrict__ work, void* __restrict__ dgate) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x;
  const int D = p.d.channels, G = p.d.gates, P = D / G;
  const ll i = e / G;
  if (i < p.offsets[0] || i >= min(p.offsets[p.d.n_segments], (ll)p.d.n_rows)) return;
  float s = 0.f;
  for (int c = 0; c < P; ++c) s += work[i * D + (e % G) * P + c];
  store1(dgate, e, p.d.gate_type, s);
}

// the rows in front of the first segment and behind the last one
__global__ void __launch_bounds__(256) scan_rest_kernel(const ll* __restrict__ offsets, ll n_seg, ll n_rows, int width, void* __restrict__ out, int type) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x, i = e / width;
  if (i < n_rows && (i < offsets[0] || i >= offsets[n_seg])) store1(out, e, type, 0.f);
}

// one thread per (row, channel): the first row of a slot takes the later ones of the same slot along, in order
__global__ void __launch_bounds__(256) step_kernel(TfGatedScan d, const void* __restrict__ gate, const void* __restrict__ x, const ll* __restrict__ slots,
                                                   ll n_slots, float* __restrict__ state, void* __restrict__ y) {
  const ll e = (ll)blockIdx.x * 256 + threadIdx.x;
  const int D = d.channels, P = D / d.gates;
  const ll r = e / D;
  if (r >= d.n_rows) return;
  const int c = (int)(e % D);
  const ll slot = slots[r];
  if (slot < 0 || slot >= n_slots) {
    if (d.zero_rest) store1(y, e, d.x_type, 0.f);
    return;
  }
  for (ll q = 0; q < r; ++q)
    if (slots[q] == slot) return;
  float h = state[slot * D + c];
  for (ll q = r; q < d.n_rows; ++q) {
    if (slots[q] != slot) continue;
    float a, b;
    gate_terms(d.form, load1(gate, q * d.ld_gate + c / P, d.gate_type), load1(x, q * d.ld_x + c, d.x_type), a, b);
    h = fmaf(a, h, b);
    store1(y, q * D + c, d.x_type, h);
  }
  state[slot * D + c] = h;
}

int rest(const TfGatedScan& d, const int64_t* offsets, int width, void* out, int type, hipStream_t stream) {
  const ll blocks = (d.n_rows * (ll)width + 255) / 256;
  TF_REQUIRE(blocks < (1ll << 31), TF_ESHAPE, "tf_gated_scan: too many rows");
  if (d.zero_rest && blocks > 0) scan_rest_kernel<<<(unsigned)blocks, 256, 0, stream>>>((const ll*)offsets, d.n_segments, d.n_rows, width, out, type);
  return TF_OK;
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

}  // namespace

extern "C" size_t tf_gated_scan_carry_floats(const TfGatedScan*) { return 0; }
extern "C" size_t tf_gated_scan_workspace_floats(const TfGatedScan* d, int32_t backward) {
  return d && backward ? (size_t)d->n_rows * d->channels : 0;
}

extern "C" int tf_gated_scan_fwd(const TfGatedScan* d, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
                                 const float* h0, void* y, float* final, float* carry, float* workspace, size_t workspace_floats, tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_scan_fwd")) return rc;
  TF_REQUIRE(offsets && (d->n_rows == 0 || (gate && x && y)), TF_EINVAL, "tf_gated_scan_fwd: null pointer");
  if (int rc = rest(*d, offsets, d->channels, y, d->x_type, (hipStream_t)stream)) return rc;
  if (d->n_segments == 0) return TF_OK;
  Scan p = {*d, gate, x, (const ll*)offsets, h0};
  const ll blocks = (d->n_segments * (ll)d->channels + 255) / 256;
  TF_REQUIRE(blocks < (1ll << 31), TF_ESHAPE, "tf_gated_scan_fwd: too many segments");
  scan_fwd_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(p, y, final);
  TF_LAUNCH_CHECK("tf_gated_scan_fwd");
  return TF_OK;
}

extern "C" int tf_gated_scan_bwd(const TfGatedScan* d, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
                                 const float* h0, const float* carry, const void* gy, const float* gfinal, void* dgate, void* dx, float* dh0, float* workspace,
                                 size_t workspace_floats, tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_scan_bwd")) return rc;
  TF_REQUIRE(offsets && (d->n_rows == 0 || (gate && x)), TF_EINVAL, "tf_gated_scan_bwd: null pointer");
  if (dx)
    if (int rc = rest(*d, offsets, d->channels, dx, d->x_type, (hipStream_t)stream)) return rc;
  if (dgate)
    if (int rc = rest(*d, offsets, d->gates, dgate, d->gate_type, (hipStream_t)stream)) return rc;
  if (d->n_segments == 0) return TF_OK;
  TF_REQUIRE(workspace_floats >= tf_gated_scan_workspace_floats(d, 1) && (d->n_rows == 0 || workspace), TF_ESHAPE, "tf_gated_scan_bwd: workspace too small");
  Scan p = {*d, gate, x, (const ll*)offsets, h0};
  const ll blocks = (d->n_segments * (ll)d->channels + 255) / 256, gblocks = (d->n_rows * (ll)d->gates + 255) / 256;
  TF_REQUIRE(blocks < (1ll << 31) && gblocks < (1ll << 31), TF_ESHAPE, "tf_gated_scan_bwd: too many rows or segments");
  scan_bwd_kernel<<<(unsigned)blocks, 256, 0, (hipStream_t)stream>>>(p, gy, gfinal, workspace, dx, dh0);
  if (dgate && gblocks > 0) scan_gate_grad_kernel<<<(unsigned)gblocks, 256, 0, (hipStream_t)stream>>>(p, workspace, dgate);
  TF_LAUNCH_CHECK("tf_gated_scan_bwd");
  return TF_OK;
}

extern "C" int tf_gated_step(const TfGatedScan* d, const void* gate, const void* x, const int64_t* slots, int64_t n_slots, float* state, void* y,
                             tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_step")) return rc;
  TF_REQUIRE(n_slots >= 0 && d->n_rows <= 65536, TF_ESHAPE, "tf_gated_step: a negative pool size, or over 65536 rows");
  if (d->n_rows == 0) return TF_OK;
  TF_REQUIRE(gate && x && slots && y && (n_slots == 0 || state), TF_EINVAL, "tf_gated_step: null pointer");
  step_kernel<<<(unsigned)((d->n_rows * (ll)d->channels + 255) / 256), 256, 0, (hipStream_t)stream>>>(*d, gate, x, (const ll*)slots, n_slots, state, y);
  TF_LAUNCH_CHECK("tf_gated_step");
  return TF_OK;
}
