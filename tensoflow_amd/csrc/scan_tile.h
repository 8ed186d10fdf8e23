// Shared by the two directions of the gated linear recurrence (scan_fwd.hip, scan_bwd.hip).
//
// h_t = a_t h_{t-1} + b_t.  The packed rows are ONE sequence to the kernels: a row that is a segment's first does not look at the row before it.
// So the work is cut into equal tiles of rows, however ragged the segments are.  A run of rows maps the state in front of it to the state behind it
// by h -> A h + B (A = prod a, B the state reached from 0), or to B alone if a segment begins in it ("closed"); two such maps join to one.
//   lane: K rows of V channels, kept in registers;  wave: 64 / CL row groups joined by shuffles;  workgroup: its waves joined through LDS;
//   tiles: each posts its (A, B) as one 64-bit word that is its own flag; the last of GRP tiles posts the group's, the last of GRP groups the state at
//   its end.  A tile finds the state in front of it from at most GRP - 1 words of its group, GRP - 1 of the groups before and one end: the only
//   chain left runs over GRP x GRP tiles a hop.
// Every input is read once, every output written once.  The words are joined in an order that the tile numbers fix, whoever came first: results repeat
// bit by bit.  A workgroup takes its tile from a counter, so the tiles that it waits for were taken by workgroups that are running or done: every wait ends.
// Bound: memory.
#pragma once
#include "tf_common.h"

namespace tfscan {

typedef long long ll;
typedef unsigned long long ull;

constexpr int K = 8;                      // consecutive rows of a lane
constexpr int GRP = 8;                    // tiles of a group, groups of a supergroup
constexpr ull EMPTY = ~0ull;              // a word that is not there yet: both halves NaNs that `clean` never lets through
constexpr unsigned CLOSED = 0xfffffffeu;  // in the place of A: B is the state, whatever came before

struct ScanArgs {
  const void *gate, *x;
  const ll *offsets, *index;
  const ull* starts;
  const float* h0;
  ll n_rows, n_seg, ld_x, ld_gate;
  int tiles, D, G, P, form, reverse, zero_rest;
  int CL, W, LP, hs, parts, slabs;  // lanes across channels, channels of a workgroup; lanes of a head, heads of a workgroup, workgroups of a head
  int narrow;                       // bytes of a wave's buffer where rows are shorter than a cache line, or 0
  int tickets;                      // distance between the counters of the slabs
  ull *words, *groups;              // [tiles][D], [tiles / GRP][D]
  unsigned *ends, *ticket;          // [tiles / GRP / GRP][D] fp32 bits
};

struct Geo {
  int V, CL, W, LP, hs, parts, slabs, nw;
  bool shared;
  ll tile_rows, tiles;
};
struct Launch {
  ScanArgs a;
  Geo g;
  unsigned blocks;
  size_t lds;
  hipStream_t stream;
};
// scan.hip
int check_desc(const TfGatedScan* d, const char* who);
Geo geometry(const TfGatedScan& d);
size_t chain_floats(const TfGatedScan& d, const Geo& g);
size_t parts_floats(const TfGatedScan& d, const Geo& g);
int prepare(const TfGatedScan& d, const char* who, const void* gate, const void* x, const int64_t* offsets, const int64_t* index, const uint64_t* starts,
            const float* h0, bool empties, float* workspace, tf_stream_t stream, const void* const* like_x, const void* like_gate, int lds_floats, Launch* out);

#define TF_SCAN_V(CALL, XT, GT, SH, WIDE)               \
  switch (L.g.V) {                                      \
    case 1: CALL(XT, GT, 1, SH, WIDE); break;           \
    case 2: CALL(XT, GT, 2, SH, WIDE); break;           \
    case 3: CALL(XT, GT, 3, SH, WIDE); break;           \
    default: CALL(XT, GT, 4, SH, WIDE); break;          \
  }
#define TF_SCAN_W(CALL, XT, GT, SH)                     \
  if (L.g.CL == 64) { TF_SCAN_V(CALL, XT, GT, SH, true) } else { TF_SCAN_V(CALL, XT, GT, SH, false) }
#define TF_SCAN_S(CALL, XT, GT)                         \
  if (L.g.shared) { TF_SCAN_W(CALL, XT, GT, true) } else { TF_SCAN_W(CALL, XT, GT, false) }
#define TF_SCAN_DISPATCH(CALL, d)                                                                       \
  if ((d).x_type == TF_TYPE_F32) { TF_SCAN_S(CALL, float, float) }                                      \
  else if ((d).x_type == TF_TYPE_F16 && (d).gate_type == TF_TYPE_F16) { TF_SCAN_S(CALL, f16, f16) } \
  else if ((d).x_type == TF_TYPE_F16) { TF_SCAN_S(CALL, f16, float) }                                \
  else if ((d).gate_type == TF_TYPE_BF16) { TF_SCAN_S(CALL, bf16, bf16) }           \
  else { TF_SCAN_S(CALL, bf16, float) }

#ifdef __HIPCC__
// compiler types: conversions are the hardware's, results rounded once, to nearest, ties to even
typedef _Float16 f16;
typedef __bf16 bf16;
template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// V neighbours of a row as they come from memory, in whole words: 16-bit values stay packed and are widened where they are used
template <typename T, int V>
struct Raw {
  static constexpr int N = (V * (int)sizeof(T) + 3) / 4;
  unsigned w[N];
  __device__ __forceinline__ float operator[](int v) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[v]);
    else return (float)__builtin_bit_cast(T, (unsigned short)(v & 1 ? w[v / 2] >> 16 : w[v / 2]));
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0;
  }
  // as if read anew: what was computed from it before is computed again, not kept beside it
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[i]));
  }
};
typedef unsigned u2 __attribute__((ext_vector_type(2)));
typedef unsigned u4 __attribute__((ext_vector_type(4)));
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> load_v(const T* p) {
  Raw<T, V> r;
  constexpr int BYTES = sizeof(T) * V;
  if constexpr (BYTES == 16) {
    const u4 q = *reinterpret_cast<const u4*>(p);
    r.w[0] = q.x, r.w[1] = q.y, r.w[2] = q.z, r.w[3] = q.w;
  } else if constexpr (BYTES == 8) {
    const u2 q = *reinterpret_cast<const u2*>(p);
    r.w[0] = q.x, r.w[1] = q.y;
  } else if constexpr (sizeof(T) == 4 || BYTES == 4) {
#pragma unroll
    for (int i = 0; i < Raw<T, V>::N; ++i) r.w[i] = reinterpret_cast<const unsigned*>(p)[i];
  } else {
    const unsigned short* s = reinterpret_cast<const unsigned short*>(p);
    r.w[0] = s[0];
    if constexpr (V == 3) r.w[0] |= (unsigned)s[1] << 16, r.w[1] = s[2];
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ Raw<T, V> round_v(const float* f) {
  Raw<T, V> r;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int v = 0; v < V; ++v) r.w[v] = __builtin_bit_cast(unsigned, f[v]);
  } else {
    r.zero();
#pragma unroll
    for (int v = 0; v < V; ++v) r.w[v / 2] |= (unsigned)__builtin_bit_cast(unsigned short, from_f<T>(f[v])) << (v & 1 ? 16 : 0);
    // beyond the compiler's sight: it would take the words apart into stores of single values
#pragma unroll
    for (int i = 0; i < Raw<T, V>::N; ++i) asm("" : "+v"(r.w[i]));
  }
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void put_v(T* p, const Raw<T, V>& r) {
  constexpr int BYTES = sizeof(T) * V;
  if constexpr (BYTES == 16) *reinterpret_cast<u4*>(p) = u4{r.w[0], r.w[1], r.w[2], r.w[3]};
  else if constexpr (BYTES == 8) *reinterpret_cast<u2*>(p) = u2{r.w[0], r.w[1]};
  else if constexpr (sizeof(T) == 4 || BYTES == 4) {
#pragma unroll
    for (int i = 0; i < Raw<T, V>::N; ++i) reinterpret_cast<unsigned*>(p)[i] = r.w[i];
  } else {
    unsigned short* s = reinterpret_cast<unsigned short*>(p);
    s[0] = (unsigned short)r.w[0];
    if constexpr (V == 3) s[1] = (unsigned short)(r.w[0] >> 16), s[2] = (unsigned short)r.w[1];
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T* p, const float* f) { put_v<T, V>(p, round_v<T, V>(f)); }

__device__ __forceinline__ unsigned clean(float f) { return f != f ? 0x7fc00000u : __float_as_uint(f); }
// exp(g) = 2^(g log2 e) on the hardware's 2^x (1 ulp): g's product is rounded once, a relative error of the result of |g| 2^-24
__device__ __forceinline__ float exp_gate(float g) { return __builtin_amdgcn_exp2f(g * 1.44269504088896341f); }

// a row's gates as ga (g of TF_GATE_ALPHA, else a): a = ga * s1 + s0, exact where nothing is to be done; fp32 ones are kept in that form
template <typename GT, int AV>
__device__ __forceinline__ void gates_kept(Raw<GT, AV>& r, int form) {
  if constexpr (sizeof(GT) == 4) {
    if (form == TF_GATE_LOG) {
#pragma unroll
      for (int v = 0; v < AV; ++v) r.w[v] = __builtin_bit_cast(unsigned, exp_gate(r[v]));
    }
  }
}
template <typename GT, int AV>
__device__ __forceinline__ void gates_of(const Raw<GT, AV>& r, int form, float (&ga)[AV]) {
#pragma unroll
  for (int v = 0; v < AV; ++v) ga[v] = r[v];
  if constexpr (sizeof(GT) == 2) {
    if (form == TF_GATE_LOG) {
#pragma unroll
      for (int v = 0; v < AV; ++v) ga[v] = exp_gate(ga[v]);
    }
  }
}

// words and ends are written and read past the caches of one XCD, each word whole: no fence orders anything else
__device__ __forceinline__ ull peek(const ull* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ unsigned peek(const unsigned* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename T>
__device__ __forceinline__ void post(T* p, T v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ ull word_of(float A, float B, bool closed) { return ((ull)(closed ? CLOSED : clean(A)) << 32) | clean(B); }

// a map of the state: h -> closed ? B : A h + B.  Whether it is closed goes by the rows alone: the same in all lanes.
struct Map {
  float A = 1.f, B = 0.f;
  bool closed = false;
};
// the n < GRP words of channel c before row `at` of D, the nearest first
struct Words {
  ull w[GRP - 1];
  __device__ __forceinline__ void ask(const ull* at, int D, int c, int n) {
#pragma unroll
    for (int i = 0; i < GRP - 1; ++i) w[i] = i < n ? peek(at - (ll)(i + 1) * D + c) : 0;
  }
  // those that are not there yet again, until they are; then joined
  __device__ __forceinline__ void join(const ull* at, int D, int c, int n, Map& m) {
    while (true) {
      bool missing = false;
#pragma unroll
      for (int i = 0; i < GRP - 1; ++i) missing |= w[i] == EMPTY;
      if (!__any(missing)) break;
      __builtin_amdgcn_s_sleep(1);
#pragma unroll
      for (int i = 0; i < GRP - 1; ++i)
        if (w[i] == EMPTY) w[i] = peek(at - (ll)(i + 1) * D + c);
    }
#pragma unroll
    for (int i = 0; i < GRP - 1; ++i) {
      if (i >= n || m.closed) break;
      const unsigned a = (unsigned)(w[i] >> 32);
      m.B = fmaf(m.A, __uint_as_float((unsigned)w[i]), m.B);
      m.closed = __builtin_amdgcn_readfirstlane(a) == CLOSED;
      m.A *= __uint_as_float(a);
    }
  }
};
// posts tile q's own map of channel c -> the state in front of it
__device__ __forceinline__ float chain(const ScanArgs& p, int q, int c, float A, float B, bool closed, bool opened) {
  const int D = p.D, iq = q % GRP, g = q / GRP, ig = g % GRP, s = g / GRP;
  ull *words = p.words + (ll)q * D, *groups = p.groups + (ll)g * D;
  unsigned* ends = p.ends + (ll)s * D;
  post(words + c, word_of(A, B, closed));
  Map m;
  m.closed = opened;
  Words w;
  if (!opened && iq) {
    w.ask(words, D, c, iq);
    w.join(words, D, c, iq, m);
  }
  if (iq == GRP - 1) post(groups + c, closed ? word_of(A, B, true) : word_of(A * m.A, fmaf(A, m.B, B), m.closed));
  unsigned e = 0;
  if (!m.closed) {
    if (s) e = peek(ends - D + c);
    if (ig) {
      w.ask(groups, D, c, ig);
      w.join(groups, D, c, ig, m);
    }
  }
  float h = m.B;
  if (!m.closed && s) {
    while (__any(e == 0xffffffffu)) {
      __builtin_amdgcn_s_sleep(1);
      e = peek(ends - D + c);
    }
    h = fmaf(m.A, __uint_as_float(e), m.B);
  }
  if (iq == GRP - 1 && ig == GRP - 1) post(ends + c, clean(closed ? B : fmaf(A, h, B)));
  return h;
}

// a lane's place: its channels (the same in all its rows) ...
template <int V, bool SHARED>
struct Lane {
  int c, g, wl, part;  // first channel, gate, lane within the head, piece of the head
  bool ok, head;       // it has channels; its head has some
  __device__ __forceinline__ Lane(const ScanArgs& p, int slab, int cl) {
    wl = 0;
    part = 0;
    if (!SHARED) {
      c = g = slab * p.W + cl * V;
      ok = c < p.D;
    } else if (p.parts == 1) {
      const int h = (unsigned)cl / (unsigned)p.LP;
      wl = cl - h * p.LP;
      g = slab * p.hs + h;
      ok = h < p.hs && g < p.G;
      c = g * p.P + wl * V;
    } else {
      g = (unsigned)slab / (unsigned)p.parts;
      part = slab - g * p.parts;
      wl = cl;
      const int w = (part * p.LP + cl) * V;
      ok = w < p.P;
      c = g * p.P + w;
    }
    head = ok || (SHARED && p.parts > 1);
    if (!ok) c = 0;
    if (!head) g = 0;
  }
};
// ... and its rows p0, p0 + step, ... in the order of the recurrence (WIDE: the same for the whole wave, kept in scalar registers).  A reversed scan
// runs over the rows tiles * T - 1 .. 0, so that tiles begin at multiples of their size in either direction.
template <bool WIDE>
struct Rows {
  ll p0, low;  // the 0-th row, the lowest one
  int step;
  unsigned valid, in;  // bit k: the k-th row is a segment's / a row
  __device__ __forceinline__ Rows(const ScanArgs& p, ll l0, ll T, ll lo, ll hi) {
    p0 = p.reverse ? p.tiles * T - 1 - l0 : l0;
    step = p.reverse ? -1 : 1;
    low = p.reverse ? p0 - (K - 1) : p0;
    valid = ordered(p, span(lo - low, hi - low));
    in = ordered(p, span(0, p.n_rows - low));
  }
  __device__ __forceinline__ static unsigned ordered(const ScanArgs& p, unsigned m) { return p.reverse ? __brev(m) >> (32 - K) : m; }
  // bits a .. b - 1 of K
  __device__ __forceinline__ static unsigned span(ll a, ll b) {
    const int f = (int)min(max(a, 0ll), (ll)K), t = (int)min(max(b, 0ll), (ll)K);
    return t > f ? ((1u << t) - 1) & ~((1u << f) - 1) : 0u;
  }
  // bit k: the k-th row is its segment's first / last in the order of the recurrence
  __device__ __forceinline__ void bits(const ScanArgs& p, ll hi, unsigned& first, unsigned& last) const {
    ull w = 0;
    if (low < p.n_rows) {
      const ll q = low >> 6, words = (p.n_rows + 63) >> 6;
      const int s = (int)(low & 63);
      w = p.starts[q] >> s;
      if (s > 64 - (K + 1) && q + 1 < words) w |= p.starts[q + 1] << (64 - s);
    }
    const unsigned f = (unsigned)w & ((1u << K) - 1);
    unsigned l = (unsigned)(w >> 1) & ((1u << K) - 1);
    const ll e = hi - 1 - low;
    if (e >= 0 && e < K) l |= 1u << e;
    first = ordered(p, p.reverse ? l : f) & valid;
    last = ordered(p, p.reverse ? f : l) & valid;
    if (WIDE) {
      first = __builtin_amdgcn_readfirstlane(first);
      last = __builtin_amdgcn_readfirstlane(last);
    }
  }
};
// the masks are tested again in every pass over the rows: held as lane masks from the first pass to the last, they fill the scalar registers
template <bool WIDE>
__device__ __forceinline__ unsigned again(unsigned m) {
  if (WIDE) asm volatile("" : "+s"(m));
  else asm volatile("" : "+v"(m));
  return m;
}
// a row of [n_seg, D]: the state of the segment that row r belongs to
template <int V>
__device__ __forceinline__ void state_of(const ScanArgs& p, const float* s, ll r, int c, float* out) {
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

// the state in front of row k: h itself, or where the segment (or what is no segment's) begins there 0 or s of its segment
template <int V, bool WIDE>
__device__ __forceinline__ void cut_at(const ScanArgs& p, int k, unsigned cut, unsigned edge, const float* s, ll r, int c, float* h) {
  if (WIDE) {
    if (cut >> k & 1) {
#pragma unroll
      for (int v = 0; v < V; ++v) h[v] = 0.f;
      if (s && (edge >> k & 1)) state_of<V>(p, s, r, c, h);
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = cut >> k & 1 ? 0.f : h[v];
    if (s && (edge >> k & 1)) state_of<V>(p, s, r, c, h);
  }
}

// The same for all rows of a lane at once, where lanes have rows of their own: row after row, each with a wait for its index and one for its state,
// the edges of short segments cost more than the rest (8000003 x 4 fp32, 23 rows a segment: 160 us, 123 with all at once).  Lanes without an edge read a place that is there.
template <bool WIDE>
__device__ __forceinline__ void segs_of(const ScanArgs& p, const Rows<WIDE>& r, unsigned edge, int (&seg)[K]) {
  ll v[K];
#pragma unroll
  for (int k = 0; k < K; ++k) v[k] = p.index[edge >> k & 1 ? r.p0 + k * r.step : 0];
#pragma unroll
  for (int k = 0; k < K; ++k) seg[k] = (edge >> k & 1) && v[k] >= 0 && v[k] < p.n_seg ? (int)v[k] : -1;
}
template <int V>
__device__ __forceinline__ void states_of(const ScanArgs& p, const float* s, const int (&seg)[K], int c, float (&out)[K][V]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int v = 0; v < V; ++v) out[k][v] = s[(ll)max(seg[k], 0) * p.D + c + v];
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

// Rows shorter than a cache line: a lane's K rows are K pieces of one line, and a load of the wave would touch 64 of them.  So the wave loads and stores
// its rows, one stretch of memory, 16 bytes a lane side by side, and turns them in LDS; a lane's rows lie 16 bytes further apart there than in
// memory, which spreads the lanes over the banks.  (8000003 x 4 fp32 compositing: 340 us with every lane at its own rows.)
__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}
template <typename T, int V>
struct Turn {
  static constexpr int NC = (K * V * (int)sizeof(T) + 15) / 16;  // 16-byte pieces of a lane, at most
  u4 piece[NC];
  int unit, magic, count;  // pieces of a lane's K rows; of the wave
  __device__ __forceinline__ Turn(int width, int RL) {
    unit = K * width * (int)sizeof(T) / 16;
    magic = (65536 + unit - 1) / unit;  // i / unit for i < 512, as unit < 128
    count = RL * unit;
  }
  __device__ __forceinline__ int place(int i) const { return (i + ((i * magic) >> 16)) * 16; }
  __device__ __forceinline__ void load(const T* rows) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < NC; ++j) piece[j] = j * 64 + lane < count ? reinterpret_cast<const u4*>(rows)[j * 64 + lane] : u4{0, 0, 0, 0};
  }
  // pieces -> the lane's rows; block: which K rows of the wave's, in memory's order
  __device__ __forceinline__ void to_rows(char* buf, int width, int block, int c, bool reverse, Raw<T, V> (&out)[K]) {
    const int lane = threadIdx.x & 63;
    wave_fence();
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (j * 64 + lane < count) *reinterpret_cast<u4*>(buf + place(j * 64 + lane)) = piece[j];
    wave_fence();
    const T* at = reinterpret_cast<const T*>(buf + block * (unit + 1) * 16) + c;
#pragma unroll
    for (int k = 0; k < K; ++k) out[k] = load_v<T, V>(at + (reverse ? K - 1 - k : k) * width);
  }
  // and back: the lane's row k
  __device__ __forceinline__ void put(char* buf, int width, int block, int c, bool reverse, int k, const Raw<T, V>& v) const {
    put_v<T, V>(reinterpret_cast<T*>(buf + block * (unit + 1) * 16) + (reverse ? K - 1 - k : k) * width + c, v);
  }
  __device__ __forceinline__ void store(const char* buf, T* rows) const {
    const int lane = threadIdx.x & 63;
    wave_fence();
#pragma unroll
    for (int j = 0; j < NC; ++j)
      if (j * 64 + lane < count) reinterpret_cast<u4*>(rows)[j * 64 + lane] = *reinterpret_cast<const u4*>(buf + place(j * 64 + lane));
  }
};

// the lane's rows as they lie in memory
template <typename T, int V, bool WIDE>
__device__ __forceinline__ void direct_rows(const T* base, ll ld, const Rows<WIDE>& r, int c, bool full, Raw<T, V> (&out)[K]) {
  if (full) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const T* row = base + (r.p0 + k * r.step) * ld;
      out[k] = load_v<T, V>(row + c);
    }
  } else {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const T* row = base + (r.p0 + k * r.step) * ld;
      out[k].zero();
      if (r.valid >> k & 1) out[k] = load_v<T, V>(row + c);
    }
  }
}

// (A, B) of a lane joined with those of the row groups before it (DOWN: behind it) in its wave; e: without its own
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
  eclosed = false;
#pragma unroll
  for (int v = 0; v < V; ++v) eB[v] = 0.f;
#pragma unroll
  for (int v = 0; v < AV; ++v) eA[v] = 1.f;
  if (p.CL == 64) return;
  const bool any = at >= p.CL;
  const bool c2 = DOWN ? __shfl_down((int)closed, p.CL) : __shfl_up((int)closed, p.CL);
  eclosed = any && c2;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const float b = DOWN ? __shfl_down(B[v], p.CL) : __shfl_up(B[v], p.CL);
    if (any) eB[v] = b;
  }
#pragma unroll
  for (int v = 0; v < AV; ++v) {
    const float a = DOWN ? __shfl_down(A[v], p.CL) : __shfl_up(A[v], p.CL);
    if (any) eA[v] = a;
  }
}

// Which job: a slab's tiles are taken in their order from the slab's counter (a counter gives 80 million tickets a second: one for all slabs would
// bound 64 x 256 tiles of 16-bit values at 5 TB/s).  Jobs behind the tiles: slab -1.
__device__ __forceinline__ int take_job(const ScanArgs& p, unsigned* s, int& slab) {
  const unsigned work = (unsigned)p.tiles * p.slabs;
  if (blockIdx.x >= work) {
    slab = -1;
    return blockIdx.x - work;
  }
  const unsigned q = blockIdx.x / (unsigned)p.slabs;
  slab = blockIdx.x - q * p.slabs;
  if (!p.ticket) return q;
  if (threadIdx.x == 0) *s = atomicAdd(p.ticket + slab * p.tickets, 1u);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(*s);
}

// The waves' (A, B) in LDS, joined by one thread for each channel; finds the state in front of the tile and puts the states in front of the waves into
// sB.  DOWN: the last wave comes first.
template <int V, bool SHARED, bool DOWN>
__device__ __forceinline__ void join_waves(const ScanArgs& p, int q, int slab, int nw, const float* sA, float* sB, const int* sclosed, bool opened, float* carry) {
  for (int t = threadIdx.x; t < p.W; t += nw * 64) {
    const Lane<V, SHARED> l(p, slab, t / V);
    if (!l.ok) continue;
    const int c = l.c + t % V;
    float h = 0.f;
    if (p.ticket) {
      float A = 1.f, B = 0.f;
      bool closed = false;
#pragma unroll 4
      for (int i = 0; i < nw; ++i) {
        const int w = DOWN ? nw - 1 - i : i;
        const float a = sA[w * p.W + t], b = sB[w * p.W + t];
        const bool cut = __builtin_amdgcn_readfirstlane(sclosed[w]);
        closed |= cut;
        B = cut ? b : fmaf(a, B, b);
        A *= a;
      }
      h = chain(p, q, c, A, B, closed, opened);
    }
    if (carry) carry[(ll)q * p.D + c] = h;
    for (int i = 0; i < nw; ++i) {
      const int w = DOWN ? nw - 1 - i : i;
      const float b = sB[w * p.W + t];
      sB[w * p.W + t] = h;
      h = sclosed[w] ? b : fmaf(sA[w * p.W + t], h, b);
    }
  }
}
#endif

}  // namespace tfscan
