// Gated linear recurrence over a packed batch of sequences, h_t = a_t h_{t-1} + b_t, its gradients and its one-token form.
//   TF_GATE_DECAY: a = g, b = x;   TF_GATE_LOG: a = exp(g), b = x;   TF_GATE_ALPHA: a = 1 - g, b = g x (compositing).
// Backward, l_t the gradient of h_t: l_t = gy_t + a_{t+1} l_{t+1}; d b_t = l_t; d a_t = l_t h_{t-1}; d h0 = a_0 l_0.
//
// The packed rows are ONE sequence to the kernels: a row that is a segment's first does not look at the row before it.  So the work is cut
// into equal tiles of rows, however ragged the segments are.  A run of rows maps the state in front of it to the state behind it by
// h -> A h + B (A = prod a, B the state reached from 0), or to B alone if a segment begins in it ("closed"); two such maps join to one.
//   lane: K rows of V channels, kept in registers;  wave: 64 / CL row groups joined by shuffles;  workgroup: its waves joined through LDS;
//   tiles: each publishes its (A, B) as one 64-bit word that is its own flag, and finds the state in front of it from the words of the tiles
//   before it in its group of GRP and the state at the end of the group before.  Every input is read once, every output written once.
// The words are joined in an order that the tile numbers fix, whoever came first: results repeat bit by bit.  A workgroup takes its tile from
// a counter, so the tiles that it waits for have been taken before it by workgroups that are running or done: every wait ends.
// Bound: memory.
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include "tf_common.h"

namespace {

typedef long long ll;
typedef unsigned long long ull;

constexpr int K = 8;                            // consecutive rows of a lane
constexpr int GRP = 16;                         // tiles whose words are joined behind one known state
constexpr ull EMPTY = ~0ull;                    // a word that is not there yet: both halves NaNs that `clean` never lets through
constexpr unsigned CLOSED = 0xfffffffeu;        // in the place of A: B is the state, whatever came before

struct ScanArgs {
  const void *gate, *x;
  const ll *offsets, *index;
  const ull* starts;
  const float* h0;
  ll n_rows, n_seg, ld_x, ld_gate, tiles;
  int D, G, P, form, reverse, zero_rest, aligned;
  int CL, W, LP, hs, parts, slabs;              // lanes across channels, channels of a workgroup; lanes of a head, heads of a workgroup, workgroups of a head
  ull* words;                                   // [tiles][D]
  unsigned* ends;                               // [tiles / GRP][D], as fp32 bits
  unsigned* ticket;
};

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
// the one rounding of a result to its type: to nearest, ties to even
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half(v); }
template <> __device__ __forceinline__ __hip_bfloat16 from_f(float v) { return __float2bfloat16(v); }

template <typename T, int V>
struct alignas((V & (V - 1)) ? sizeof(T) : sizeof(T) * V) Vec {
  T v[V];
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_v(const T* p, bool aligned) {
  if (aligned) return *reinterpret_cast<const Vec<T, V>*>(p);
  Vec<T, V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = p[v];
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float* f, bool aligned) {
  Vec<T, V> r;
#pragma unroll
  for (int v = 0; v < V; ++v) r.v[v] = from_f<T>(f[v]);
  if (aligned) {
    *reinterpret_cast<Vec<T, V>*>(p) = r;
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) p[v] = r.v[v];
  }
}

__device__ __forceinline__ unsigned clean(float f) { return f != f ? 0x7fc00000u : __float_as_uint(f); }
// exp(g) = 2^(g log2 e) on the hardware's 2^x (1 ulp): g's product is rounded once, a relative error of the result of |g| 2^-24
__device__ __forceinline__ float exp_gate(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504088896341f); }

// words and ends are written and read past the caches of one XCD, each word whole: no fence orders anything else
__device__ __forceinline__ ull peek(const ull* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned peek(const unsigned* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ void post(T* p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// the state in front of the q-th tile of channel c
__device__ __forceinline__ float state_before(const ScanArgs& p, ll q, int c) {
  const ll g0 = q - q % GRP;
  ull w[GRP - 1];
#pragma unroll
  for (int m = 0; m < GRP - 1; ++m)
    if (q - 1 - m >= g0) w[m] = peek(p.words + (q - 1 - m) * p.D + c);
  unsigned e = g0 ? peek(p.ends + (g0 / GRP - 1) * p.D + c) : 0u;
  float A = 1.f, B = 0.f;
#pragma unroll
  for (int m = 0; m < GRP - 1; ++m) {
    if (q - 1 - m < g0) break;
    while (w[m] == EMPTY) {
      __builtin_amdgcn_s_sleep(1);
      w[m] = peek(p.words + (q - 1 - m) * p.D + c);
    }
    B = fmaf(A, __uint_as_float((unsigned)w[m]), B);
    if ((unsigned)(w[m] >> 32) == CLOSED) return B;
    A *= __uint_as_float((unsigned)(w[m] >> 32));
  }
  if (!g0) return B;
  while (e == 0xffffffffu) {
    __builtin_amdgcn_s_sleep(1);
    e = peek(p.ends + (g0 / GRP - 1) * p.D + c);
  }
  return fmaf(A, __uint_as_float(e), B);
}

// a lane's place: its channels (the same in all its rows) ...
template <int V, bool SHARED>
struct Lane {
  int c, g, wl, part;  // first channel, gate, lane within the head, piece of the head
  bool ok;
  __device__ Lane(const ScanArgs& p, int slab, int cl) {
    wl = 0;
    part = 0;
    if (!SHARED) {
      c = g = slab * p.W + cl * V;
      ok = c < p.D;
    } else if (p.parts == 1) {
      const int h = cl / p.LP;
      wl = cl - h * p.LP;
      g = slab * p.hs + h;
      ok = h < p.hs && g < p.G;
      c = g * p.P + wl * V;
    } else {
      g = slab / p.parts;
      part = slab - g * p.parts;
      wl = cl;
      const int w = (part * p.LP + cl) * V;
      ok = w < p.P;
      c = g * p.P + w;
    }
    if (!ok) c = g = 0;
  }
};
// ... and its rows, in the order of the recurrence: bit k of first / last / valid for its k-th row
struct Rows {
  ll p0;     // the 0-th row
  int step;  // to the next one
  unsigned first, last, valid, in;
  __device__ Rows(const ScanArgs& p, ll l0, ll lo, ll hi) {
    const ll n = p.n_rows;
    p0 = p.reverse ? n - 1 - l0 : l0;
    step = p.reverse ? -1 : 1;
    const ll b = p.reverse ? p0 - (K - 1) : p0;  // the lowest of the rows b .. b + K - 1
    ull bits = 0;
    if (b < n && b + K >= 0) {
      const ll q = b < 0 ? 0 : b, w = q >> 6, words = (n + 63) >> 6;
      const int s = (int)(q & 63);
      bits = p.starts[w] >> s;
      if (s && w + 1 < words) bits |= p.starts[w + 1] << (64 - s);
      bits <<= q - b;
    }
    unsigned f = 0, l = 0, v = 0, i = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const ll r = b + k;
      const unsigned one = 1u << k;
      if (r >= 0 && r < n) i |= one;
      if (r >= lo && r < hi) v |= one;
      if (bits >> k & 1) f |= one;
      if ((bits >> (k + 1) & 1) || r + 1 == hi) l |= one;
    }
    first = p.reverse ? __brev(l) >> (32 - K) : f;
    last = p.reverse ? __brev(f) >> (32 - K) : l;
    valid = p.reverse ? __brev(v) >> (32 - K) : v;
    in = p.reverse ? __brev(i) >> (32 - K) : i;
    first &= valid;
    last &= valid;
  }
};

// a row of [n_seg, D]: the state of the segment that row r belongs to
template <int V>
__device__ __forceinline__ void state_of(const ScanArgs& p, const float* s, ll r, int c, float* out) {
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = 0.f;
  if (!s) return;
  const ll seg = p.index[r];
  if (seg < 0 || seg >= p.n_seg) return;
#pragma unroll
  for (int v = 0; v < V; ++v) out[v] = s[seg * p.D + c + v];
}
template <int V>
__device__ __forceinline__ void put_state(const ScanArgs& p, float* s, ll r, int c, const float* in) {
  const ll seg = p.index[r];
  if (seg < 0 || seg >= p.n_seg) return;
#pragma unroll
  for (int v = 0; v < V; ++v) s[seg * p.D + c + v] = in[v];
}

// segments without rows hand `from` (or 0) on to `to`: a wave looks at 64 of them and copies row after row
__device__ __forceinline__ void empty_segments(const ScanArgs& p, ll wave, const float* from, float* to) {
  const int lane = threadIdx.x & 63;
  const ll s = wave * 64 + lane;
  ull todo = __ballot(s < p.n_seg && p.offsets[s + 1] <= p.offsets[s]);
  while (todo) {
    const ll e = wave * 64 + __ffsll((long long)todo) - 1;
    todo &= todo - 1;
    for (int c = lane; c < p.D; c += 64) to[e * p.D + c] = from ? from[e * p.D + c] : 0.f;
  }
}

template <typename XT, typename GT, int V, bool SHARED>
struct Tile {
  static constexpr int AV = SHARED ? 1 : V;
  Vec<XT, V> rx[K];
  Vec<GT, AV> rg[K];
  __device__ __forceinline__ void load(const ScanArgs& p, const Rows& r, const Lane<V, SHARED>& l, bool fast) {
    const XT* x = static_cast<const XT*>(p.x) + r.p0 * p.ld_x + l.c;
    const GT* g = static_cast<const GT*>(p.gate) + r.p0 * p.ld_gate + l.g;
    const ll sx = r.step * p.ld_x, sg = r.step * p.ld_gate;
    if (fast) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        rx[k] = load_v<XT, V>(x + k * sx, true);
        rg[k] = load_v<GT, AV>(g + k * sg, true);
      }
    } else {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        if (r.valid >> k & 1) {
          rx[k] = load_v<XT, V>(x + k * sx, false);
          rg[k] = load_v<GT, AV>(g + k * sg, false);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) rx[k].v[v] = from_f<XT>(0.f);
#pragma unroll
          for (int v = 0; v < AV; ++v) rg[k].v[v] = from_f<GT>(0.f);
        }
      }
    }
  }
};

// (A, B) of a lane joined with those of the row groups before it (DOWN: behind it) in its wave -> of all of them, without its own
template <int V, int AV, bool DOWN>
__device__ __forceinline__ void wave_join(const ScanArgs& p, float (&A)[AV], float (&B)[V], bool& closed, float (&eA)[AV], float (&eB)[V], bool& eclosed) {
  const int lane = threadIdx.x & 63;
  const int at = DOWN ? 63 - lane : lane;
  for (int o = p.CL; o < 64; o <<= 1) {
    const bool c2 = DOWN ? __shfl_down((int)closed, o) : __shfl_up((int)closed, o);
    const bool take = at >= o && !closed;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float b = DOWN ? __shfl_down(B[v], o) : __shfl_up(B[v], o);
      if (take) B[v] = fmaf(A[AV == 1 ? 0 : v], b, B[v]);
    }
#pragma unroll
    for (int v = 0; v < AV; ++v) {
      const float a = DOWN ? __shfl_down(A[v], o) : __shfl_up(A[v], o);
      if (take) A[v] *= a;
    }
    if (take) closed = c2;
  }
  eclosed = DOWN ? __shfl_down((int)closed, p.CL) : __shfl_up((int)closed, p.CL);
  const bool none = at < p.CL;
  if (none) eclosed = false;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    eB[v] = DOWN ? __shfl_down(B[v], p.CL) : __shfl_up(B[v], p.CL);
    if (none) eB[v] = 0.f;
  }
#pragma unroll
  for (int v = 0; v < AV; ++v) {
    eA[v] = DOWN ? __shfl_down(A[v], p.CL) : __shfl_up(A[v], p.CL);
    if (none) eA[v] = 1.f;
  }
}

// which tile: taken from the counter where tiles wait for each other
__device__ __forceinline__ ll take_ticket(const ScanArgs& p, unsigned* s) {
  if (!p.ticket) return blockIdx.x;
  if (threadIdx.x == 0) *s = atomicAdd(p.ticket, 1u);
  __syncthreads();
  return *s;
}

// the waves' (A, B) in LDS, joined by one thread for each channel: publishes the tile's own, finds the state in front of it and puts the states in
// front of the waves into sB.  order: the wave that comes i-th.
template <int V, bool SHARED, bool DOWN>
__device__ __forceinline__ void join_waves(const ScanArgs& p, ll q, int slab, int nw, float* sA, float* sB, const int* sclosed, bool opened, float* carry) {
  const bool chain = p.ticket != nullptr;
  for (int t = threadIdx.x; t < p.W; t += nw * 64) {
    const Lane<V, SHARED> l(p, slab, t / V);
    if (!l.ok) continue;
    const int c = l.c + t % V;
    float A = 1.f, B = 0.f;
    bool closed = false;
    for (int i = 0; i < nw; ++i) {
      const int w = DOWN ? nw - 1 - i : i;
      if (sclosed[w]) {
        B = sB[w * p.W + t];
        closed = true;
      } else {
        B = fmaf(sA[w * p.W + t], B, sB[w * p.W + t]);
        A *= sA[w * p.W + t];
      }
    }
    float h = 0.f;
    if (chain) {
      post(p.words + q * p.D + c, ((ull)(closed ? CLOSED : clean(A)) << 32) | clean(B));
      if (!opened) h = state_before(p, q, c);
    }
    if (carry) carry[q * p.D + c] = h;
    for (int i = 0; i < nw; ++i) {
      const int w = DOWN ? nw - 1 - i : i;
      const float b = sB[w * p.W + t];
      sB[w * p.W + t] = h;
      h = sclosed[w] ? b : fmaf(sA[w * p.W + t], h, b);
    }
    if (chain && q % GRP == GRP - 1) post(p.ends + (q / GRP) * p.D + c, clean(h));
  }
}

template <typename XT, typename GT, int V, bool SHARED>
__global__ void __launch_bounds__(512) scan_fwd_kernel(ScanArgs p, XT* __restrict__ y, float* __restrict__ final, float* __restrict__ carry) {
  extern __shared__ float smem[];
  __shared__ unsigned s_ticket;
  __shared__ int s_closed[8], s_opened;
  constexpr int AV = SHARED ? 1 : V;
  const int nw = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float *sA = smem, *sB = smem + nw * p.W;
  const ll job = take_ticket(p, &s_ticket), work = p.tiles * p.slabs;
  if (job >= work) {
    empty_segments(p, (job - work) * nw + wave, p.h0, final);
    return;
  }
  const ll q = job / p.slabs;
  const int slab = (int)(job - q * p.slabs);
  const int cl = lane & (p.CL - 1), rl = lane / p.CL, RL = 64 / p.CL;
  const ll T = (ll)nw * RL * K, lo = p.offsets[0], hi = p.offsets[p.n_seg];
  const Lane<V, SHARED> l(p, slab, cl);
  const ll l0 = q * T + (wave * RL + rl) * K, a0 = p.reverse ? p.n_rows - (q + 1) * T : q * T;
  const Rows r(p, l0, lo, hi);
  const bool fast = p.aligned && a0 >= lo && a0 + T <= hi;
  Tile<XT, GT, V, SHARED> t;
  t.load(p, r, l, fast);
  // a and b
  float a[K][AV], b[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) b[k][v] = to_f(t.rx[k].v[v]);
#pragma unroll
    for (int v = 0; v < AV; ++v) a[k][v] = to_f(t.rg[k].v[v]);
  }
  if (p.form == TF_GATE_LOG) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int v = 0; v < AV; ++v) a[k][v] = exp_gate(a[k][v]);
  } else if (p.form == TF_GATE_ALPHA) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int v = 0; v < V; ++v) b[k][v] *= a[k][AV == 1 ? 0 : v];
#pragma unroll
      for (int v = 0; v < AV; ++v) a[k][v] = 1.f - a[k][v];
    }
  }
  float A[AV], B[V], eA[AV], eB[V];
  bool closed = false, eclosed;
#pragma unroll
  for (int v = 0; v < AV; ++v) A[v] = 1.f;
#pragma unroll
  for (int v = 0; v < V; ++v) B[v] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!(r.valid >> k & 1)) {
      closed = true;
#pragma unroll
      for (int v = 0; v < V; ++v) B[v] = 0.f;
      continue;
    }
    if (r.first >> k & 1) {
      closed = true;
      state_of<V>(p, p.h0, r.p0 + k * r.step, l.c, B);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) B[v] = fmaf(a[k][AV == 1 ? 0 : v], B[v], b[k][v]);
#pragma unroll
    for (int v = 0; v < AV; ++v) A[v] *= a[k][v];
  }
  wave_join<V, AV, false>(p, A, B, closed, eA, eB, eclosed);
  if (rl == RL - 1) {
#pragma unroll
    for (int v = 0; v < V; ++v) {
      sA[wave * p.W + cl * V + v] = A[AV == 1 ? 0 : v];
      sB[wave * p.W + cl * V + v] = B[v];
    }
    if (cl == 0) s_closed[wave] = closed;
  }
  if (threadIdx.x == 0) s_opened = (r.first & 1) || !(r.valid & 1);
  __syncthreads();
  join_waves<V, SHARED, false>(p, q, slab, nw, sA, sB, s_closed, s_opened, carry);
  __syncthreads();
  float h[V];
#pragma unroll
  for (int v = 0; v < V; ++v) h[v] = eclosed ? eB[v] : fmaf(eA[AV == 1 ? 0 : v], sB[wave * p.W + cl * V + v], eB[v]);
  if (!l.ok) return;
  XT* out = y + r.p0 * p.D + l.c;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const ll at = r.p0 + k * r.step;
    if (!(r.valid >> k & 1)) {
      if (p.zero_rest && (r.in >> k & 1)) {
        const float z[V] = {};
        store_v<XT, V>(y + at * p.D + l.c, z, false);
      }
      continue;
    }
    if (r.first >> k & 1) state_of<V>(p, p.h0, at, l.c, h);
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = fmaf(a[k][AV == 1 ? 0 : v], h[v], b[k][v]);
    store_v<XT, V>(out + (ll)k * r.step * p.D, h, p.aligned);
    if (final && (r.last >> k & 1)) put_state<V>(p, final, at, l.c, h);
  }
}

// The states again from the state in front of the tile that the forward pass kept; then, in the other order, m = a l, what a row hands to the
// row before it: a segment's last row has gfinal in its place, so a tile that holds a last row is closed.
template <typename XT, typename GT, int V, bool SHARED>
__global__ void __launch_bounds__(512) scan_bwd_kernel(ScanArgs p, const float* __restrict__ carry, const XT* __restrict__ gy, const float* __restrict__ gfinal,
                                                       GT* __restrict__ dgate, float* __restrict__ dgate_parts, XT* __restrict__ dx, float* __restrict__ dh0) {
  extern __shared__ float smem[];
  __shared__ unsigned s_ticket;
  __shared__ int s_closed[8], s_mclosed[8], s_opened;
  constexpr int AV = SHARED ? 1 : V;
  const int nw = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  float *sA = smem, *sB = sA + nw * p.W, *sP = sB + nw * p.W, *sQ = sP + nw * p.W;
  const ll job = take_ticket(p, &s_ticket), work = p.tiles * p.slabs;
  if (job >= work) {
    empty_segments(p, (job - work) * nw + wave, gfinal, dh0);
    return;
  }
  const ll qd = job / p.slabs, q = p.tiles - 1 - qd;  // the tiles from the last to the first
  const int slab = (int)(job - qd * p.slabs);
  const int cl = lane & (p.CL - 1), rl = lane / p.CL, RL = 64 / p.CL;
  const ll T = (ll)nw * RL * K, lo = p.offsets[0], hi = p.offsets[p.n_seg];
  const Lane<V, SHARED> l(p, slab, cl);
  const ll l0 = q * T + (wave * RL + rl) * K, a0 = p.reverse ? p.n_rows - (q + 1) * T : q * T;
  const Rows r(p, l0, lo, hi);
  const bool fast = p.aligned && a0 >= lo && a0 + T <= hi;
  Tile<XT, GT, V, SHARED> t;
  Vec<XT, V> rgy[K];
  t.load(p, r, l, fast);
  if (gy && fast) {
#pragma unroll
    for (int k = 0; k < K; ++k) rgy[k] = load_v<XT, V>(gy + (r.p0 + k * r.step) * p.D + l.c, true);
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (gy && (r.valid >> k & 1)) {
        rgy[k] = load_v<XT, V>(gy + (r.p0 + k * r.step) * p.D + l.c, false);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) rgy[k].v[v] = from_f<XT>(0.f);
      }
    }
  }
  // ga: a, or g itself where a = 1 - g; a = ga * s1 + s0 and b = x * (ga or 1), both exact where nothing is to be done
  const bool alpha = p.form == TF_GATE_ALPHA;
  const float s1 = alpha ? -1.f : 1.f, s0 = alpha ? 1.f : 0.f;
  float ga[K][AV], x[K][V], g[K][V], before[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k) {
#pragma unroll
    for (int v = 0; v < V; ++v) x[k][v] = to_f(t.rx[k].v[v]);
#pragma unroll
    for (int v = 0; v < V; ++v) g[k][v] = to_f(rgy[k].v[v]);
#pragma unroll
    for (int v = 0; v < AV; ++v) ga[k][v] = to_f(t.rg[k].v[v]);
  }
  if (p.form == TF_GATE_LOG) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int v = 0; v < AV; ++v) ga[k][v] = exp_gate(ga[k][v]);
  }
  float A[AV], B[V], eA[AV], eB[V], P[AV], Q[V], eP[AV], eQ[V];
  bool closed = false, eclosed, mclosed = false, emclosed;
#pragma unroll
  for (int v = 0; v < AV; ++v) A[v] = P[v] = 1.f;
#pragma unroll
  for (int v = 0; v < V; ++v) B[v] = Q[v] = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!(r.valid >> k & 1)) {
      closed = true;
#pragma unroll
      for (int v = 0; v < V; ++v) B[v] = 0.f;
      continue;
    }
    if (r.first >> k & 1) {
      closed = true;
      state_of<V>(p, p.h0, r.p0 + k * r.step, l.c, B);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float gav = ga[k][AV == 1 ? 0 : v];
      B[v] = fmaf(fmaf(gav, s1, s0), B[v], alpha ? gav * x[k][v] : x[k][v]);
    }
#pragma unroll
    for (int v = 0; v < AV; ++v) A[v] *= fmaf(ga[k][v], s1, s0);
  }
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    if (!(r.valid >> k & 1)) {
      mclosed = true;
#pragma unroll
      for (int v = 0; v < V; ++v) Q[v] = 0.f;
      continue;
    }
    if (r.last >> k & 1) {
      mclosed = true;
      state_of<V>(p, gfinal, r.p0 + k * r.step, l.c, Q);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) Q[v] = fmaf(ga[k][AV == 1 ? 0 : v], s1, s0) * (g[k][v] + Q[v]);
#pragma unroll
    for (int v = 0; v < AV; ++v) P[v] *= fmaf(ga[k][v], s1, s0);
  }
  wave_join<V, AV, false>(p, A, B, closed, eA, eB, eclosed);
  wave_join<V, AV, true>(p, P, Q, mclosed, eP, eQ, emclosed);
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
  if (threadIdx.x == blockDim.x - 1) s_opened = (r.last >> (K - 1) & 1) || !(r.valid >> (K - 1) & 1);
  __syncthreads();
  for (int i = threadIdx.x; i < p.W; i += nw * 64) {
    const Lane<V, SHARED> ln(p, slab, i / V);
    if (!ln.ok) continue;
    float h = carry[q * p.D + ln.c + i % V];
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
    h[v] = eclosed ? eB[v] : fmaf(eA[AV == 1 ? 0 : v], sB[wave * p.W + cl * V + v], eB[v]);
    m[v] = emclosed ? eQ[v] : fmaf(eP[AV == 1 ? 0 : v], sQ[wave * p.W + cl * V + v], eQ[v]);
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if ((r.first >> k & 1) || !(r.valid >> k & 1)) state_of<V>(p, (r.valid >> k & 1) ? p.h0 : nullptr, r.p0 + k * r.step, l.c, h);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float gav = ga[k][AV == 1 ? 0 : v];
      before[k][v] = h[v];
      h[v] = fmaf(fmaf(gav, s1, s0), h[v], alpha ? gav * x[k][v] : x[k][v]);
    }
  }
#pragma unroll
  for (int k = K - 1; k >= 0; --k) {
    const ll at = r.p0 + k * r.step;
    const bool valid = r.valid >> k & 1, in = r.in >> k & 1;
    float d[V], o[V];
    if (valid && (r.last >> k & 1)) state_of<V>(p, gfinal, at, l.c, m);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const float gav = ga[k][AV == 1 ? 0 : v], lam = valid ? g[k][v] + m[v] : 0.f;
      o[v] = alpha ? gav * lam : lam;
      d[v] = valid ? lam * (alpha ? x[k][v] - before[k][v] : p.form == TF_GATE_LOG ? gav * before[k][v] : before[k][v]) : 0.f;
      m[v] = fmaf(gav, s1, s0) * lam;
    }
    const bool write = l.ok && (valid || (p.zero_rest && in));
    if (dx && write) store_v<XT, V>(dx + at * p.D + l.c, o, p.aligned);
    if (dh0 && l.ok && (r.first >> k & 1)) put_state<V>(p, dh0, at, l.c, m);
    if (dgate) {
      if (!SHARED) {
        if (write) store_v<GT, V>(dgate + at * p.G + l.c, d, p.aligned);
      } else {
        float s = 0.f;
#pragma unroll
        for (int v = 0; v < V; ++v) s += d[v];
        if (!l.ok) s = 0.f;
        for (int o2 = 1; o2 < p.LP; o2 <<= 1) {
          const float z = __shfl_down(s, o2);
          if (l.wl + o2 < p.LP) s += z;
        }
        if (write && l.wl == 0) {
          if (dgate_parts) dgate_parts[((ll)l.part * p.n_rows + at) * p.G + l.g] = s;
          else dgate[at * p.G + l.g] = from_f<GT>(s);
        }
      }
    }
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

__global__ void __launch_bounds__(256) scan_clear_kernel(ull* __restrict__ words, ll n, unsigned* __restrict__ ticket) {
  const ll i = (ll)blockIdx.x * 256 + threadIdx.x;
  if (i < n) words[i] = EMPTY;
  if (i == 0) *ticket = 0;
}

// A workgroup is a row and 256 V of its channels.  The first row of a slot takes the later ones of the same slot along, in order; the others leave.
template <typename XT, typename GT, int V, bool SHARED>
__global__ void __launch_bounds__(256) step_kernel(TfGatedScan d, int aligned, const GT* __restrict__ gate, const XT* __restrict__ x, const ll* __restrict__ slots,
                                                   ll n_slots, float* __restrict__ state, XT* __restrict__ y) {
  constexpr int AV = SHARED ? 1 : V;
  const int D = d.channels, P = D / d.gates, n = (int)d.n_rows, r = blockIdx.y, c = (blockIdx.x * 256 + threadIdx.x) * V;
  const bool mine = c < D;
  const ll slot = slots[r];
  if (slot < 0 || slot >= n_slots) {
    const float z[V] = {};
    if (d.zero_rest && mine) store_v<XT, V>(y + (ll)r * D + c, z, aligned);
    return;
  }
  const ll g = SHARED ? c / P : c;
  Vec<XT, V> rx;
  Vec<GT, AV> rg;
  Vec<float, V> h;
  if (mine) {  // asked for before the search, which needs none of it
    rx = load_v<XT, V>(x + r * d.ld_x + c, aligned);
    rg = load_v<GT, AV>(gate + r * d.ld_gate + g, aligned);
    h = load_v<float, V>(state + slot * D + c, aligned);
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
      rx = load_v<XT, V>(x + q * d.ld_x + c, aligned);
      rg = load_v<GT, AV>(gate + q * d.ld_gate + g, aligned);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = to_f(rg.v[AV == 1 ? 0 : v]), b = to_f(rx.v[v]);
      if (d.form == TF_GATE_LOG) a = exp_gate(a);
      if (d.form == TF_GATE_ALPHA) b *= a, a = 1.f - a;
      h.v[v] = fmaf(a, h.v[v], b);
    }
    store_v<XT, V>(y + (ll)q * D + c, h.v, aligned);
  }
  store_v<float, V>(state + slot * D + c, h.v, aligned);
}

// ------------------------------------------------------------------------------------------------ host
struct Geo {
  int V, CL, W, LP, hs, parts, slabs, nw;
  bool shared;
  ll tile_rows, tiles;
};
int pow2_from(int n) {
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
  g.nw = 8;
  while (g.nw > 1 && ((d.n_rows + g.nw * wave_rows - 1) / (g.nw * wave_rows)) * g.slabs < 512) g.nw >>= 1;
  for (int w = 1; w <= 8; w <<= 1)
    if (d.n_rows <= w * wave_rows && w > g.nw) g.nw = w;
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
size_t chain_floats(const TfGatedScan& d, const Geo& g) {
  return g.tiles > 1 ? 2 * (size_t)g.tiles * d.channels + ((size_t)(g.tiles / GRP) * d.channels + 1) / 2 * 2 + 2 : 0;
}
size_t parts_floats(const TfGatedScan& d, const Geo& g) { return g.shared && g.parts > 1 ? (size_t)g.parts * d.n_rows * d.gates : 0; }

bool fits(const void* p, size_t bytes) { return ((size_t)p & (bytes - 1)) == 0; }

struct Launch {
  ScanArgs a;
  Geo g;
  unsigned blocks;
  size_t lds;
  hipStream_t stream;
};

// shared by both directions: arguments, chain memory cleared, grid
int prepare(const TfGatedScan& d, const char* who, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
            const float* h0, bool empties, float* workspace, tf_stream_t stream, bool others_aligned, Launch* out) {
  const Geo g = geometry(d);
  const size_t xs = d.x_type == TF_TYPE_F32 ? 4 : 2, gs = d.gate_type == TF_TYPE_F32 ? 4 : 2;
  const int vx = g.V == 3 ? 1 : g.V, vg = g.shared ? 1 : vx;
  ScanArgs a = {gate, x, (const ll*)offsets, (const ll*)index, (const ull*)starts, h0, d.n_rows, d.n_segments, d.ld_x, d.ld_gate, g.tiles, d.channels, d.gates,
                d.channels / d.gates, d.form, d.reverse ? 1 : 0, d.zero_rest ? 1 : 0, 0, g.CL, g.W, g.LP, g.hs, g.parts, g.slabs, nullptr, nullptr, nullptr};
  a.aligned = others_aligned && fits(x, vx * xs) && fits(gate, vg * gs) && d.ld_x % vx == 0 && d.ld_gate % vg == 0;
  const ll rest = empties ? (d.n_segments + 64ll * g.nw - 1) / (64ll * g.nw) : 0, blocks = g.tiles * g.slabs + rest;
  TF_REQUIRE(blocks < (1ll << 31) - 1, TF_ESHAPE, "%s: too many rows", who);
  hipStream_t st = (hipStream_t)stream;
  if (g.tiles > 1) {
    a.words = reinterpret_cast<ull*>(workspace);
    a.ends = reinterpret_cast<unsigned*>(a.words + g.tiles * d.channels);
    const ll n = (ll)(chain_floats(d, g) / 2);
    a.ticket = reinterpret_cast<unsigned*>(a.words + n - 1);
    scan_clear_kernel<<<(unsigned)((n - 1 + 255) / 256), 256, 0, st>>>(a.words, n - 1, a.ticket);
  }
  *out = {a, g, (unsigned)blocks, 0, st};
  return TF_OK;
}

template <typename XT, typename GT, int V, bool SHARED>
void launch_fwd(const Launch& L, void* y, float* final, float* carry) {
  scan_fwd_kernel<XT, GT, V, SHARED><<<L.blocks, L.g.nw * 64, (size_t)L.g.nw * L.g.W * 2 * sizeof(float), L.stream>>>(L.a, static_cast<XT*>(y), final, carry);
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
template <typename XT, typename GT, int V, bool SHARED>
void launch_bwd(const Launch& L, const BwdPtrs& b) {
  scan_bwd_kernel<XT, GT, V, SHARED><<<L.blocks, L.g.nw * 64, (size_t)L.g.nw * L.g.W * 4 * sizeof(float), L.stream>>>(
      L.a, b.carry, static_cast<const XT*>(b.gy), b.gfinal, static_cast<GT*>(b.dgate), b.parts, static_cast<XT*>(b.dx), b.dh0);
}

#define TF_SCAN_V(CALL, XT, GT, SH)                     \
  switch (L.g.V) {                                      \
    case 1: CALL(XT, GT, 1, SH); break;                 \
    case 2: CALL(XT, GT, 2, SH); break;                 \
    case 3: CALL(XT, GT, 3, SH); break;                 \
    default: CALL(XT, GT, 4, SH); break;                \
  }
#define TF_SCAN_S(CALL, XT, GT)                         \
  if (L.g.shared) { TF_SCAN_V(CALL, XT, GT, true) } else { TF_SCAN_V(CALL, XT, GT, false) }
#define TF_SCAN_DISPATCH(CALL, d)                                                                       \
  if ((d).x_type == TF_TYPE_F32) { TF_SCAN_S(CALL, float, float) }                                      \
  else if ((d).x_type == TF_TYPE_F16 && (d).gate_type == TF_TYPE_F16) { TF_SCAN_S(CALL, __half, __half) } \
  else if ((d).x_type == TF_TYPE_F16) { TF_SCAN_S(CALL, __half, float) }                                \
  else if ((d).gate_type == TF_TYPE_BF16) { TF_SCAN_S(CALL, __hip_bfloat16, __hip_bfloat16) }           \
  else { TF_SCAN_S(CALL, __hip_bfloat16, float) }

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

extern "C" int tf_gated_scan_fwd(const TfGatedScan* d, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
                                 const float* h0, void* y, float* final, float* carry, float* workspace, size_t workspace_floats, tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_scan_fwd")) return rc;
  TF_REQUIRE(offsets && (d->n_rows == 0 || (gate && x && y && starts)), TF_EINVAL, "tf_gated_scan_fwd: null pointer");
  TF_REQUIRE(d->n_rows == 0 || index || (!h0 && !final), TF_EINVAL, "tf_gated_scan_fwd: h0 and final need an index");
  const size_t need = tf_gated_scan_workspace_floats(d, 0);
  TF_REQUIRE(workspace_floats >= need && (!need || (workspace && fits(workspace, 8))), TF_ESHAPE, "tf_gated_scan_fwd: workspace too small, or not aligned to 8 bytes");
  Launch L;
  const Geo g = geometry(*d);
  const int vx = g.V == 3 ? 1 : g.V;
  if (int rc = prepare(*d, "tf_gated_scan_fwd", gate, x, offsets, index, starts, h0, final != nullptr, workspace, stream,
                       fits(y, vx * (d->x_type == TF_TYPE_F32 ? 4 : 2)), &L))
    return rc;
  if (L.blocks) {
#define CALL(XT, GT, V, SH) launch_fwd<XT, GT, V, SH>(L, y, final, carry)
    TF_SCAN_DISPATCH(CALL, *d)
#undef CALL
  }
  TF_LAUNCH_CHECK("tf_gated_scan_fwd");
  return TF_OK;
}

extern "C" int tf_gated_scan_bwd(const TfGatedScan* d, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
                                 const float* h0, const float* carry, const void* gy, const float* gfinal, void* dgate, void* dx, float* dh0, float* workspace,
                                 size_t workspace_floats, tf_stream_t stream) {
  if (int rc = check_desc(d, "tf_gated_scan_bwd")) return rc;
  TF_REQUIRE(offsets && (d->n_rows == 0 || (gate && x && starts && carry)), TF_EINVAL, "tf_gated_scan_bwd: null pointer");
  TF_REQUIRE(d->n_rows == 0 || index || (!h0 && !gfinal && !dh0), TF_EINVAL, "tf_gated_scan_bwd: h0 and final need an index");
  const size_t need = tf_gated_scan_workspace_floats(d, 1);
  TF_REQUIRE(workspace_floats >= need && (!need || (workspace && fits(workspace, 8))), TF_ESHAPE, "tf_gated_scan_bwd: workspace too small, or not aligned to 8 bytes");
  Launch L;
  const Geo g = geometry(*d);
  const size_t vx = (g.V == 3 ? 1 : g.V) * (d->x_type == TF_TYPE_F32 ? 4 : 2), vg = g.shared ? 1 : (g.V == 3 ? 1 : g.V) * (d->gate_type == TF_TYPE_F32 ? 4 : 2);
  if (int rc = prepare(*d, "tf_gated_scan_bwd", gate, x, offsets, index, starts, h0, dh0 != nullptr, workspace, stream,
                       (!gy || fits(gy, vx)) && (!dx || fits(dx, vx)) && (!dgate || fits(dgate, vg)), &L))
    return rc;
  const BwdPtrs b = {carry, gy, gfinal, dgate, parts_floats(*d, g) ? workspace + chain_floats(*d, g) : nullptr, dx, dh0};
  const ll pblocks = b.parts && dgate ? (d->n_rows * (ll)d->gates + 255) / 256 : 0;
  TF_REQUIRE(pblocks < (1ll << 31), TF_ESHAPE, "tf_gated_scan_bwd: too many rows");
  if (L.blocks) {
#define CALL(XT, GT, V, SH) launch_bwd<XT, GT, V, SH>(L, b)
    TF_SCAN_DISPATCH(CALL, *d)
#undef CALL
  }
  if (pblocks) {
    hipStream_t st = (hipStream_t)stream;
#define PARTS(GT) scan_gate_parts_kernel<GT><<<(unsigned)pblocks, 256, 0, st>>>(b.parts, (const ll*)offsets, d->n_segments, d->n_rows, d->gates, g.parts, d->zero_rest, static_cast<GT*>(dgate))
    if (d->gate_type == TF_TYPE_F32) PARTS(float);
    else if (d->gate_type == TF_TYPE_F16) PARTS(__half);
    else PARTS(__hip_bfloat16);
#undef PARTS
  }
  TF_LAUNCH_CHECK("tf_gated_scan_bwd");
  return TF_OK;
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
  const int V = unit % 4 == 0 && d->n_rows * d->channels >= 65536 ? 4 : 1;
  const size_t xs = d->x_type == TF_TYPE_F32 ? 4 : 2, gs = d->gate_type == TF_TYPE_F32 ? 4 : 2;
  const int vg = shared ? 1 : V;
  const int aligned = fits(x, V * xs) && fits(y, V * xs) && fits(gate, vg * gs) && fits(state, V * 4) && (d->n_rows == 1 || (d->ld_x % V == 0 && d->ld_gate % vg == 0));
  const dim3 grid((unsigned)((d->channels + 256 * V - 1) / (256 * V)), (unsigned)d->n_rows);
  hipStream_t st = (hipStream_t)stream;
#define STEP(XT, GT, VV, SH) step_kernel<XT, GT, VV, SH><<<grid, 256, 0, st>>>(*d, aligned, static_cast<const GT*>(gate), static_cast<const XT*>(x), (const ll*)slots, n_slots, state, static_cast<XT*>(y))
#define STEP_V(XT, GT)                                                            \
  if (V == 4) { if (shared) STEP(XT, GT, 4, true); else STEP(XT, GT, 4, false); } \
  else { if (shared) STEP(XT, GT, 1, true); else STEP(XT, GT, 1, false); }
  if (d->x_type == TF_TYPE_F32) { STEP_V(float, float) }
  else if (d->x_type == TF_TYPE_F16 && d->gate_type == TF_TYPE_F16) { STEP_V(__half, __half) }
  else if (d->x_type == TF_TYPE_F16) { STEP_V(__half, float) }
  else if (d->gate_type == TF_TYPE_BF16) { STEP_V(__hip_bfloat16, __hip_bfloat16) }
  else { STEP_V(__hip_bfloat16, float) }
#undef STEP_V
#undef STEP
  TF_LAUNCH_CHECK("tf_gated_step");
  return TF_OK;
}
