// Element-wise gated linear recurrence over [rows, T, D] tensors, dense or packed, forward, backward and one token:
//   h_t = e^{g_t} h_{t-1} + x_t,  y_t = h_t                                    (h_0 the initial state, g log-decays)
//   dh_t = dy_t + e^{g_{t+1}} dh_{t+1},  dx_t = dh_t,  dg_t = e^{g_t} h_{t-1} dh_t,  dh_0 = e^{g_1} dh_1
// No products to speak of: every pass is bound by the bytes of its tensors ([8, 4096, 2048] bf16: forward 90-97 us for 403 MB, 4.2-4.5
// TB/s, backward 131-135 for 671 MB, 5.0-5.1 TB/s; a copy reaches 4.97).  A workgroup owns 128 bytes of channels of one row and walks
// its tokens in tiles: a thread holds four channels of R consecutive tokens and reduces them to a pair (A, H), the map h -> A h + H;
// pairs are scanned over the token groups of a wave by lane swaps, and the eight waves' pairs are chained through LDS by one lane per
// channel, which carries the state from tile to tile.  The loads of the next tile are in flight meanwhile.  (Eight channels of four
// tokens a thread, scanned over eight groups by shuffles, were bound by the scan: 4.1 TB/s at [8, 4096, 2048] bf16, the same with
// twice the loads in flight.)  Everything between loads and stores is fp32.  The backward pass reads x again instead of y, which is
// rounded: the forward pass leaves a state every 128 tokens (fp32, 1 / 128 of the elements), so the states
// behind dg are the unrounded ones.
// Where rows and channels give too few workgroups every tile (of 128 tokens) has a workgroup of its own: it publishes its pair, folds
// those before it and goes on from there, all tensors still read once (a first launch for the pairs of segments and a second one
// that read everything again took 352 us for [1, 65536, 2048] with fp32 gates, 229 this way).  Workgroups of one row and channel
// tile take their tiles from a counter, so a tile is waited for only by workgroups that started after its own; it publishes before it
// waits.  Every 32nd tile publishes the pair of all 32 as soon as it has the others', every 1024th the state behind it, and a tile goes
// on from the last such state through the pairs of 32 and of one in the order of time: the same sums in the same order whatever the
// timing, results are the same from run to run.  (With states every 32 tiles each was a wait for the one before: 3.7 us in a row.)
#include "lnx_common.h"
#include "mma_tiles.h"
#include "packed_slots.h"

namespace {

constexpr int THREADS = 512, N = 4, TILE = 256;  // tokens of a tile
constexpr int CTHREADS = 256, CTILE = 128, GROUP = 32, ANCHOR = GROUP * 32;  // where every tile has a workgroup; tiles of a common pair, between states
constexpr int KEPT = 128;  // tokens between the states that the forward pass leaves for the backward pass
// By element type: threads side by side in a row, so that a row of a workgroup is 128 bytes; its channels; tokens per thread (what the
// backward pass's registers take)
template <typename T> struct Shape {
  static constexpr int COLS = sizeof(T) == 2 ? 16 : 8, C = COLS * N, R = TILE * COLS / THREADS;
  static_assert(R == CTILE * COLS / CTHREADS, "both forms hold as many tokens a thread");
};

// Four consecutive elements as they lie in memory
template <typename E, bool VEC> struct Raw {
  typename Vec4<E>::V v;
  __device__ __forceinline__ void load(const E* p, int left) {
    if (VEC) v = *reinterpret_cast<const typename Vec4<E>::V*>(p);
    else
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = i < left ? p[i] : from_f32<E>(0.f);
  }
  __device__ __forceinline__ void zero() { v = typename Vec4<E>::V{}; }
  __device__ __forceinline__ float get(int i) const { return to_f32(v[i]); }
};

template <bool VEC, typename E> __device__ __forceinline__ void put(E* p, const float (&f)[N], int left) {
  if (VEC) store4(p, floatx4{f[0], f[1], f[2], f[3]});
  else
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < left) p[i] = from_f32<E>(f[i]);
}

struct Args {
  const void *x, *g, *dy;
  int64_t xb, xt, gb, gt, yb, yt;  // strides of a row and of a token, in elements; yb, yt: of dy
  const float *s0, *ds;
  const int32_t* cu;
  void *y, *dx, *dg;
  float *sT, *d0, *kept;
  uint64_t *pairs, *sums;  // [slots of CTILE tokens][D], (A, H) of a tile, [slots of GROUP tiles][D], of GROUP tiles; all bits set: not there yet
  uint32_t* anchors;       // [slots of ANCHOR tiles][D], the state behind ANCHOR, 2 ANCHOR, ... tiles of a row; likewise
  uint32_t* counters;      // [rows][channel tiles]: tiles taken
  int T, D, ctiles;
  bool packed;
};

// What a workgroup works on: row, its channels, its tiles
template <typename T> struct Place {
  int row, len, ntile, c0, c, left;  // c0: the workgroup's first channel, c: this thread's
  int64_t tok, slot;  // first token in a packed batch (0 otherwise); first kept state
  // The first slot of the row where each holds `size` tokens
  __device__ __forceinline__ int64_t slot_of(const Args& a, int size) const {
    return a.packed ? packed_slot((int)tok, row, size) : (int64_t)row * (((int64_t)a.T + size - 1) / size);
  }
  __device__ __forceinline__ Place(const Args& a, int row_, int ct, int tile) {
    row = row_;
    if (a.packed) {
      const int first = seq_first(a.cu, row, a.T);
      len = seq_end(a.cu, row, a.T) - first;
      tok = first;
    } else {
      len = a.T;
      tok = 0;
    }
    slot = slot_of(a, KEPT);
    ntile = (int)(((int64_t)len + tile - 1) / tile);
    c0 = ct * Shape<T>::C;
    c = c0 + (threadIdx.x & (Shape<T>::COLS - 1)) * N;
    left = a.D - c;
  }
  // Token `first` of the row: the wave's pointer and the lane's bytes from there, so that addresses are formed in scalar registers
  template <typename E> __device__ __forceinline__ const char* at(const void* p, int64_t b, int64_t t, int64_t first) const {
    return static_cast<const char*>(p) + (row * b + (tok + first) * t) * (int64_t)sizeof(E);
  }
  template <typename E> __device__ __forceinline__ unsigned lane(int64_t t, int token) const { return (unsigned)((token * (int)t + c) * (int)sizeof(E)); }
};
template <typename E> __device__ __forceinline__ const E* elems(const char* p, unsigned off) { return reinterpret_cast<const E*>(p + off); }
template <typename E> __device__ __forceinline__ E* elems(char* p, unsigned off) { return reinterpret_cast<E*>(p + off); }

// (a, h): a thread's pair.  Afterwards the wave's pair, and in (ea, eh) that of the wave's groups (16 lanes each, or 8) before this
// one, upwards or downwards in time.
template <bool UP> __device__ __forceinline__ void scan16(float& a, float& h, float& ea, float& eh, int lane) {
  const auto a16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(a), false, false);  // even groups' values, odd groups'
  const auto h16 = __builtin_amdgcn_permlane16_swap(__float_as_uint(h), __float_as_uint(h), false, false);
  const float a1 = __uint_as_float(UP ? a16[0] : a16[1]), h1 = __uint_as_float(UP ? h16[0] : h16[1]);  // the first of two groups
  const float a2 = __uint_as_float(UP ? a16[1] : a16[0]), h2 = __uint_as_float(UP ? h16[1] : h16[0]);
  const float ap = a1 * a2, hp = a2 * h1 + h2;
  const bool second = ((lane >> 4) & 1) == (UP ? 1 : 0);
  ea = second ? a1 : 1.f;
  eh = second ? h1 : 0.f;
  const auto a32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(ap), __float_as_uint(ap), false, false);  // the lower half's, the upper half's
  const auto h32 = __builtin_amdgcn_permlane32_swap(__float_as_uint(hp), __float_as_uint(hp), false, false);
  const float A1 = __uint_as_float(UP ? a32[0] : a32[1]), H1 = __uint_as_float(UP ? h32[0] : h32[1]);
  const float A2 = __uint_as_float(UP ? a32[1] : a32[0]), H2 = __uint_as_float(UP ? h32[1] : h32[0]);
  a = A1 * A2;
  h = A2 * H1 + H2;
  if ((lane >> 5) == (UP ? 1 : 0)) {
    eh += ea * H1;
    ea *= A1;
  }
}

template <int COLS, bool UP> __device__ __forceinline__ void scan_wave(float& a, float& h, float& ea, float& eh, int lane) {
  if (COLS == 16) return scan16<UP>(a, h, ea, eh, lane);
  const float ao = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(a), 0x128, 0xF, 0xF, true));  // row_ror:8, the other group of 16 lanes
  const float ho = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(h), 0x128, 0xF, 0xF, true));
  const bool second = ((lane >> 3) & 1) == (UP ? 1 : 0);
  const float own_a = a, own_h = h;
  a = own_a * ao;
  h = second ? own_a * ho + own_h : ao * own_h + ho;
  scan16<UP>(a, h, ea, eh, lane);
  if (second) {  // before this group: what came before the two, then the other one
    eh = ao * eh + ho;
    ea *= ao;
  }
}

// The waves' pairs and the states entering the waves, by channel of the workgroup
template <int COLS, int WAVES> struct Waves {
  static constexpr int C = COLS * N;
  float A[WAVES][C], H[WAVES][C], in[WAVES][C];
  __device__ __forceinline__ void leave(const float (&a)[N], const float (&h)[N], int lane, int wave) {
    if (lane < COLS) {
      store4(&A[wave][lane * N], floatx4{a[0], a[1], a[2], a[3]});
      store4(&H[wave][lane * N], floatx4{h[0], h[1], h[2], h[3]});
    }
  }
  // one lane per channel: the state entering each wave, `carry` from before the tile to behind it
  template <bool UP> __device__ __forceinline__ void chain(int c, float& carry) {
    float a[WAVES], h[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) a[w] = A[w][c], h[w] = H[w][c];
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const int w = UP ? k : WAVES - 1 - k;
      in[w][c] = carry;
      carry = a[w] * carry + h[w];
    }
  }
  // one lane per channel: the tile's pair
  template <bool UP> __device__ __forceinline__ void total(int c, float& A_, float& H_) const {
    A_ = 1.f;
    H_ = 0.f;
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const int w = UP ? k : WAVES - 1 - k;
      H_ = A[w][c] * H_ + H[w][c];
      A_ *= A[w][c];
    }
  }
  // the state entering this thread's tokens
  __device__ __forceinline__ void enter(const float (&ea)[N], const float (&eh)[N], float (&s)[N], int lane, int wave) const {
    const floatx4 from = load4(&in[wave][(lane & (COLS - 1)) * N]);
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = ea[i] * from[i] + eh[i];
  }
};

// What a thread holds of a tile: the vectors of its R tokens from `x` and `g` on
template <typename T, typename G, bool VEC> struct Tokens {
  static constexpr int R = Shape<T>::R;
  Raw<T, VEC> x[R];
  Raw<G, VEC> g[R];
};

// ---- words that other workgroups wait for ----
constexpr uint32_t EMPTY = 0xffffffffu, QUIET = 0x7fc00000u;
// (Waits end by themselves, see above; a bound keeps a fault elsewhere from holding the GPU: the result is NaN then.)
constexpr int MOST_POLLS = 1 << 22;
__device__ __forceinline__ uint32_t word(float x) {
  const uint32_t u = __float_as_uint(x);
  return u == EMPTY ? QUIET : u;
}
__device__ __forceinline__ uint64_t peek(const uint64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ uint32_t peek(const uint32_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void publish(uint64_t* p, float A, float H) {
  __hip_atomic_store(p, (uint64_t)word(A) << 32 | word(H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void publish(uint32_t* p, float x) { __hip_atomic_store(p, word(x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
template <typename W> __device__ __forceinline__ W await(const W* p, W v) {
  for (int n = 0; (uint32_t)v == EMPTY && n < MOST_POLLS; ++n) {
    __builtin_amdgcn_s_sleep(1);
    v = peek(p);
  }
  return v;
}

// (A, H) := the n maps of `p` (D apart) behind it: one lane per channel
__device__ __forceinline__ void fold(float& A, float& H, const uint64_t* p, int n, int D) {
  for (int i = 0; i < n; i += 8) {
    uint64_t v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = i + u < n ? peek(p + (int64_t)(i + u) * D) : (uint64_t)__float_as_uint(1.f) << 32;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      if (i + u < n) v[u] = await(p + (int64_t)(i + u) * D, v[u]);
      const float a = __uint_as_float((uint32_t)(v[u] >> 32));
      H = a * H + __uint_as_float((uint32_t)v[u]);
      A *= a;
    }
  }
}
// The state before the j-th of ntile tiles (counted from where the recurrence starts), from `begin` before the first; (A, H) is the
// tile's pair.  Leaves what others wait for before it waits for what comes before the tile's group.  One lane per channel.
template <typename P> __device__ __forceinline__ float state_before(const Args& a, const P& p, int j, int chan, float begin, float A, float H) {
  const int base = j / GROUP * GROUP, top = j / ANCHOR * ANCHOR, ntile = p.ntile;
  uint64_t* pairs = a.pairs + p.slot_of(a, CTILE) * a.D + chan;
  uint64_t* sums = a.sums + p.slot_of(a, CTILE * GROUP) * a.D + chan;
  if (j + 1 < ntile) publish(pairs + (int64_t)j * a.D, A, H);
  float Ag = 1.f, Hg = 0.f;
  fold(Ag, Hg, pairs + (int64_t)base * a.D, j - base, a.D);
  if (j - base == GROUP - 1 && j + 1 < ntile) publish(sums + (int64_t)(j / GROUP) * a.D, A * Ag, A * Hg + H);
  float state = begin;
  if (top) {
    const uint32_t* at = a.anchors + (p.slot_of(a, CTILE * ANCHOR) + top / ANCHOR - 1) * a.D + chan;
    state = __uint_as_float(await(at, peek(at)));
  }
  float unused = 1.f;
  fold(unused, state, sums + (int64_t)(top / GROUP) * a.D, (base - top) / GROUP, a.D);
  return Ag * state + Hg;
}
template <typename P> __device__ __forceinline__ void leave_state(const Args& a, const P& p, int j, int chan, float state) {
  if ((j + 1) % ANCHOR == 0 && j + 1 < p.ntile) publish(a.anchors + (p.slot_of(a, CTILE * ANCHOR) + (j + 1) / ANCHOR - 1) * a.D + chan, state);
}
// The row of this workgroup; its channel tile is blockIdx % ctiles
__device__ __forceinline__ int chain_row(const Args& a, int rows) {
  const int unit = blockIdx.x / a.ctiles;
  return a.packed ? packed_owner(a.cu, rows, a.T, CTILE, unit) : unit % rows;
}
// The tile of this workgroup: the next one of its row and channels
__device__ __forceinline__ int take_tile(const Args& a, int group) {
  __shared__ int tile;
  if (threadIdx.x == 0) tile = (int)__hip_atomic_fetch_add(a.counters + group, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(tile);
}
__global__ __launch_bounds__(256) void linrec_clear_kernel(uint32_t* words, int64_t n, uint32_t* counters, int groups) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (4 * i + 3 < n) *reinterpret_cast<uint4*>(words + 4 * i) = uint4{EMPTY, EMPTY, EMPTY, EMPTY};
  else
    for (int64_t k = 4 * i; k < n; ++k) words[k] = EMPTY;
  if (i < groups) counters[i] = 0;
}

// The pointers of a forward pass at token `first` of the row, and a lane's bytes from there
template <typename T, typename G, bool VEC> struct Forward {
  static constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  const char *x, *g;
  char* y;
  unsigned xo, go, yo;
  int64_t xs, gs, ys;
  int tr;
  __device__ __forceinline__ Forward(const Args& a, const Place<T>& p, int64_t first) {
    const int64_t row_b = a.packed ? 0 : 1;  // a packed batch is one row
    tr = threadIdx.x / COLS;
    x = p.template at<T>(a.x, row_b * a.xb, a.xt, first);
    g = p.template at<G>(a.g, row_b * a.gb, a.gt, first);
    y = const_cast<char*>(p.template at<T>(a.y, row_b * a.T * a.D, a.D, first));
    xo = p.template lane<T>(a.xt, tr * R), go = p.template lane<G>(a.gt, tr * R), yo = p.template lane<T>(a.D, tr * R);
    xs = a.xt * (int64_t)sizeof(T), gs = a.gt * (int64_t)sizeof(G), ys = a.D * (int64_t)sizeof(T);
  }
  // `there`: tokens of the row from the tile's first on
  __device__ __forceinline__ void fetch(Tokens<T, G, VEC>& in, const Place<T>& p, const Args& a, int64_t there, int tile) const {
    if (there >= tile && p.c0 + C <= a.D) {
#pragma unroll
      for (int u = 0; u < R; ++u) in.x[u].load(elems<T>(x + u * xs, xo), N), in.g[u].load(elems<G>(g + u * gs, go), N);
    } else {
#pragma unroll
      for (int u = 0; u < R; ++u) {
        in.x[u].zero();
        in.g[u].zero();
        if (tr * R + u < there && p.left > 0) in.x[u].load(elems<T>(x + u * xs, xo), p.left), in.g[u].load(elems<G>(g + u * gs, go), p.left);
      }
    }
  }
  __device__ __forceinline__ void finish(const Place<T>& p, const Args& a, int64_t there, int tile, float (&h)[N], const float (&e)[R][N], const float (&xv)[R][N]) const {
    const bool whole = there >= tile && p.c0 + C <= a.D;
#pragma unroll
    for (int u = 0; u < R; ++u) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] = e[u][i] * h[i] + xv[u][i];
      if (whole || (tr * R + u < there && p.left > 0)) put<VEC>(elems<T>(y + u * ys, yo), h, p.left);
    }
  }
};
// A thread's factors and inputs, and its pair
template <typename T, typename G, bool VEC>
__device__ __forceinline__ void reduce_forward(const Tokens<T, G, VEC>& in, float (&e)[Shape<T>::R][N], float (&xv)[Shape<T>::R][N], float (&A)[N], float (&H)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) A[i] = 1.f, H[i] = 0.f;
#pragma unroll
  for (int u = 0; u < Shape<T>::R; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      e[u][i] = __expf(in.g[u].get(i));  // 1 behind the end: the state stands
      xv[u][i] = in.x[u].get(i);
      H[i] = e[u][i] * H[i] + xv[u][i];
      A[i] *= e[u][i];
    }
}

template <typename T, typename G, bool VEC> __global__ __launch_bounds__(THREADS) void linrec_fwd_kernel(Args a) {
  constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  __shared__ Waves<COLS, 8> ws;
  const Place<T> p(a, blockIdx.x / a.ctiles, blockIdx.x % a.ctiles, TILE);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  // the chain's lanes: one channel each
  const int chan = p.c0 + lane;
  const bool chains = wave == 0 && lane < C, in_chan = chains && chan < a.D;
  float carry = in_chan && a.s0 ? a.s0[(int64_t)p.row * a.D + chan] : 0.f;
  Forward<T, G, VEC> f(a, p, 0);
  Tokens<T, G, VEC> in;
  if (p.ntile) f.fetch(in, p, a, p.len, TILE);
  for (int tile = 0; tile < p.ntile; ++tile) {
    const int64_t there = p.len - (int64_t)tile * TILE;
    float e[R][N], xv[R][N], A[N], H[N], ea[N], eh[N], h[N];
    reduce_forward<T, G, VEC>(in, e, xv, A, H);
    f.x += TILE * f.xs;
    f.g += TILE * f.gs;
    if (tile + 1 < p.ntile) f.fetch(in, p, a, there - TILE, TILE);
#pragma unroll
    for (int i = 0; i < N; ++i) scan_wave<COLS, true>(A[i], H[i], ea[i], eh[i], lane);
    ws.leave(A, H, lane, wave);
    lds_barrier();
    if (chains) {
      ws.template chain<true>(lane, carry);
      if (a.kept && in_chan) {
#pragma unroll
        for (int k = 0; k < TILE / KEPT; ++k)
          if (k * KEPT < there) a.kept[(p.slot + tile * (TILE / KEPT) + k) * a.D + chan] = ws.in[k * 8 * KEPT / TILE][lane];
      }
    }
    lds_barrier();
    ws.enter(ea, eh, h, lane, wave);
    f.finish(p, a, there, TILE, h, e, xv);
    f.y += TILE * f.ys;
  }
  if (in_chan) a.sT[(int64_t)p.row * a.D + chan] = carry;
}

template <typename T, typename G, bool VEC> __global__ __launch_bounds__(CTHREADS) void linrec_fwd_chain_kernel(Args a, int rows) {
  constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  __shared__ Waves<COLS, 4> ws;
  const int row = chain_row(a, rows), ct = blockIdx.x % a.ctiles, j = take_tile(a, row * a.ctiles + ct);
  const Place<T> p(a, row, ct, CTILE);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, chan = p.c0 + lane;
  const bool in_chan = wave == 0 && lane < C && chan < a.D;
  const int64_t row_c = (int64_t)p.row * a.D + chan;
  if (j >= p.ntile) {
    if (j == 0 && in_chan) a.sT[row_c] = a.s0 ? a.s0[row_c] : 0.f;  // no tokens at all
    return;
  }
  const int64_t first = (int64_t)j * CTILE, there = p.len - first;
  const Forward<T, G, VEC> f(a, p, first);
  Tokens<T, G, VEC> in;
  f.fetch(in, p, a, there, CTILE);
  float e[R][N], xv[R][N], A[N], H[N], ea[N], eh[N], h[N];
  reduce_forward<T, G, VEC>(in, e, xv, A, H);
#pragma unroll
  for (int i = 0; i < N; ++i) scan_wave<COLS, true>(A[i], H[i], ea[i], eh[i], lane);
  ws.leave(A, H, lane, wave);
  lds_barrier();
  if (in_chan) {
    float At, Ht;
    ws.template total<true>(lane, At, Ht);
    float carry = state_before(a, p, j, chan, a.s0 ? a.s0[row_c] : 0.f, At, Ht);
    if (a.kept) a.kept[(p.slot + j) * a.D + chan] = carry;
    ws.template chain<true>(lane, carry);
    leave_state(a, p, j, chan, carry);
    if (j + 1 == p.ntile) a.sT[row_c] = carry;
  }
  lds_barrier();
  ws.enter(ea, eh, h, lane, wave);
  f.finish(p, a, there, CTILE, h, e, xv);
}

// The pointers of a backward pass
template <typename T, typename G, bool VEC> struct Backward {
  static constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  const char *x, *g, *dy;
  char *dx, *dg;
  unsigned xo, go, yo, dxo, dgo;
  int64_t xs, gs, ys, dxs, dgs;
  int tr;
  __device__ __forceinline__ Backward(const Args& a, const Place<T>& p, int64_t first) {
    const int64_t row_b = a.packed ? 0 : 1;
    tr = threadIdx.x / COLS;
    x = p.template at<T>(a.x, row_b * a.xb, a.xt, first);
    g = p.template at<G>(a.g, row_b * a.gb, a.gt, first);
    dy = p.template at<T>(a.dy, row_b * a.yb, a.yt, first);
    dx = const_cast<char*>(p.template at<T>(a.dx, row_b * a.T * a.D, a.D, first));
    dg = const_cast<char*>(p.template at<G>(a.dg, row_b * a.T * a.D, a.D, first));
    xo = p.template lane<T>(a.xt, tr * R), go = p.template lane<G>(a.gt, tr * R), yo = p.template lane<T>(a.yt, tr * R);
    dxo = p.template lane<T>(a.D, tr * R), dgo = p.template lane<G>(a.D, tr * R);
    xs = a.xt * (int64_t)sizeof(T), gs = a.gt * (int64_t)sizeof(G), ys = a.yt * (int64_t)sizeof(T), dxs = a.D * (int64_t)sizeof(T), dgs = a.D * (int64_t)sizeof(G);
  }
  __device__ __forceinline__ void fetch(Tokens<T, G, VEC>& in, Raw<T, VEC> (&yr)[R], const Place<T>& p, const Args& a, int64_t there, int tile) const {
    if (there >= tile && p.c0 + C <= a.D) {
#pragma unroll
      for (int u = 0; u < R; ++u) in.x[u].load(elems<T>(x + u * xs, xo), N), in.g[u].load(elems<G>(g + u * gs, go), N);
      if (a.dy) {
#pragma unroll
        for (int u = 0; u < R; ++u) yr[u].load(elems<T>(dy + u * ys, yo), N);
      } else {
#pragma unroll
        for (int u = 0; u < R; ++u) yr[u].zero();
      }
    } else {
#pragma unroll
      for (int u = 0; u < R; ++u) {
        in.x[u].zero();
        in.g[u].zero();
        yr[u].zero();
        if (tr * R + u < there && p.left > 0) {
          in.x[u].load(elems<T>(x + u * xs, xo), p.left);
          if (a.dy) yr[u].load(elems<T>(dy + u * ys, yo), p.left);
          in.g[u].load(elems<G>(g + u * gs, go), p.left);
        }
      }
    }
  }
  // h: the state before this thread's tokens, o: e^g dh of the token behind them
  __device__ __forceinline__ void finish(const Place<T>& p, const Args& a, int64_t there, int tile, float (&h)[N], float (&o)[N], const float (&e)[R][N],
                                         const Raw<T, VEC> (&xk)[R], const Raw<T, VEC> (&yk)[R]) const {
    const bool whole = there >= tile && p.c0 + C <= a.D;
    float hb[R][N];
#pragma unroll
    for (int u = 0; u < R; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) hb[u][i] = h[i], h[i] = e[u][i] * h[i] + xk[u].get(i);
#pragma unroll
    for (int u = R - 1; u >= 0; --u) {
      float dh[N], dgv[N];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        dh[i] = yk[u].get(i) + o[i];
        o[i] = e[u][i] * dh[i];
        dgv[i] = hb[u][i] * o[i];
      }
      if (whole || (tr * R + u < there && p.left > 0)) {
        put<VEC>(elems<T>(dx + u * dxs, dxo), dh, p.left);
        put<VEC>(elems<G>(dg + u * dgs, dgo), dgv, p.left);
      }
    }
  }
};
// A thread's factors and its two pairs: of the gradients backwards in time (o is e^{g_{t+1}} dh_{t+1}), of the states forwards
template <typename T, typename G, bool VEC>
__device__ __forceinline__ void reduce_backward(const Tokens<T, G, VEC>& in, const Raw<T, VEC> (&yr)[Shape<T>::R], float (&e)[Shape<T>::R][N], float (&A)[N], float (&H)[N],
                                                float (&Af)[N], float (&Hf)[N]) {
  constexpr int R = Shape<T>::R;
#pragma unroll
  for (int i = 0; i < N; ++i) A[i] = 1.f, H[i] = 0.f, Hf[i] = 0.f;
#pragma unroll
  for (int u = R - 1; u >= 0; --u)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      e[u][i] = __expf(in.g[u].get(i));
      H[i] = e[u][i] * (yr[u].get(i) + H[i]);
      A[i] *= e[u][i];
    }
#pragma unroll
  for (int u = 0; u < R; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) Hf[i] = e[u][i] * Hf[i] + in.x[u].get(i);
#pragma unroll
  for (int i = 0; i < N; ++i) Af[i] = A[i];
}

template <typename T, typename G, bool VEC> __global__ __launch_bounds__(THREADS) void linrec_bwd_kernel(Args a) {
  constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  __shared__ Waves<COLS, 8> ws, wf;
  const Place<T> p(a, blockIdx.x / a.ctiles, blockIdx.x % a.ctiles, TILE);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int chan = p.c0 + lane;  // wave 0 chains the gradients, wave 1 the states
  const bool mine = lane < C && chan < a.D, grads = wave == 0 && lane < C, states = wave == 1 && lane < C;
  float carry = grads && mine && a.ds ? a.ds[(int64_t)p.row * a.D + chan] : 0.f, start = 0.f;
  Backward<T, G, VEC> f(a, p, (int64_t)(p.ntile - 1) * TILE);  // the last tile
  Tokens<T, G, VEC> in;
  Raw<T, VEC> yr[R];
  const auto fetch = [&](int tile) {
    if (states && mine) start = a.kept[(p.slot + (int64_t)tile * (TILE / KEPT)) * a.D + chan];
    f.fetch(in, yr, p, a, p.len - (int64_t)tile * TILE, TILE);
  };
  if (p.ntile) fetch(p.ntile - 1);
  for (int tile = p.ntile - 1; tile >= 0; --tile) {
    float e[R][N], A[N], H[N], ea[N], eh[N], Af[N], Hf[N], fa[N], fh[N], h[N], o[N];
    reduce_backward<T, G, VEC>(in, yr, e, A, H, Af, Hf);
    Raw<T, VEC> xk[R], yk[R];
#pragma unroll
    for (int u = 0; u < R; ++u) xk[u] = in.x[u], yk[u] = yr[u];
    float from = start;
    f.x -= TILE * f.xs;
    f.g -= TILE * f.gs;
    f.dy -= TILE * f.ys;
    if (tile > 0) fetch(tile - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      scan_wave<COLS, true>(Af[i], Hf[i], fa[i], fh[i], lane);
      scan_wave<COLS, false>(A[i], H[i], ea[i], eh[i], lane);
    }
    wf.leave(Af, Hf, lane, wave);
    ws.leave(A, H, lane, wave);
    lds_barrier();
    if (grads) ws.template chain<false>(lane, carry);
    if (states) wf.template chain<true>(lane, from);
    lds_barrier();
    wf.enter(fa, fh, h, lane, wave);
    ws.enter(ea, eh, o, lane, wave);
    f.finish(p, a, p.len - (int64_t)tile * TILE, TILE, h, o, e, xk, yk);
    f.dx -= TILE * f.dxs;
    f.dg -= TILE * f.dgs;
  }
  if (grads && mine && a.d0) a.d0[(int64_t)p.row * a.D + chan] = carry;
}

template <typename T, typename G, bool VEC> __global__ __launch_bounds__(CTHREADS) void linrec_bwd_chain_kernel(Args a, int rows) {
  constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  __shared__ Waves<COLS, 4> ws, wf;
  const int row = chain_row(a, rows), ct = blockIdx.x % a.ctiles, j = take_tile(a, row * a.ctiles + ct);
  const Place<T> p(a, row, ct, CTILE);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, chan = p.c0 + lane;
  const bool mine = lane < C && chan < a.D, grads = wave == 0 && mine, states = wave == 1 && mine;
  const int64_t row_c = (int64_t)p.row * a.D + chan;
  if (j >= p.ntile) {
    if (j == 0 && grads && a.d0) a.d0[row_c] = a.ds ? a.ds[row_c] : 0.f;
    return;
  }
  const int tile = p.ntile - 1 - j;
  const int64_t first = (int64_t)tile * CTILE, there = p.len - first;
  const Backward<T, G, VEC> f(a, p, first);
  Tokens<T, G, VEC> in;
  Raw<T, VEC> yr[R];
  f.fetch(in, yr, p, a, there, CTILE);
  float e[R][N], A[N], H[N], ea[N], eh[N], Af[N], Hf[N], fa[N], fh[N], h[N], o[N];
  reduce_backward<T, G, VEC>(in, yr, e, A, H, Af, Hf);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    scan_wave<COLS, true>(Af[i], Hf[i], fa[i], fh[i], lane);
    scan_wave<COLS, false>(A[i], H[i], ea[i], eh[i], lane);
  }
  wf.leave(Af, Hf, lane, wave);
  ws.leave(A, H, lane, wave);
  lds_barrier();
  if (grads) {
    float At, Ht;
    ws.template total<false>(lane, At, Ht);
    float carry = state_before(a, p, j, chan, a.ds ? a.ds[row_c] : 0.f, At, Ht);
    ws.template chain<false>(lane, carry);
    leave_state(a, p, j, chan, carry);
    if (tile == 0 && a.d0) a.d0[row_c] = carry;
  }
  if (states) {
    float from = a.kept[(p.slot + tile) * a.D + chan];
    wf.template chain<true>(lane, from);
  }
  lds_barrier();
  wf.enter(fa, fh, h, lane, wave);
  ws.enter(ea, eh, o, lane, wave);
  f.finish(p, a, there, CTILE, h, o, e, in.x, yr);
}

// One token: four elements a thread, or one where the vectors do not fit
template <typename T, typename G, int W> __global__ __launch_bounds__(256) void linrec_step_kernel(const T* x, const G* g, const float* s, T* y, float* s_out, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * W;
  if (i >= n) return;
  if (W == 4) {
    const floatx4 xv = load4(x + i), gv = load4(g + i), sv = load4(s + i);
    floatx4 h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __expf(gv[e]) * sv[e] + xv[e];
    store4(y + i, h);
    store4(s_out + i, h);
  } else {
    const float h = __expf(to_f32(g[i])) * s[i] + to_f32(x[i]);
    y[i] = from_f32<T>(h);
    s_out[i] = h;
  }
}

constexpr int64_t MAX_STRIDE = 4 << 20, MAX_GRID = 0xffffffff;  // threads of a launch
int rows_of(const lnx_linrec_args* a) { return a->nseq ? a->nseq : a->B; }
int channel_tiles(const lnx_linrec_args* a) {
  const int c = a->dtype == LNX_BF16 ? Shape<bf16_t>::C : Shape<float>::C;
  return (int)(((int64_t)a->D + c - 1) / c);
}

// Slots of `size` tokens in all rows
int64_t slots_of(const lnx_linrec_args* a, int64_t size) { return a->nseq ? a->T / size + a->nseq : a->B * ((a->T + size - 1) / size); }
// Whether every tile has a workgroup of its own: where walking the rows would leave a third of the chip without work.  With 256 rows and
// channel tiles both forms move bytes at the same rate forwards and the walk is 13 % faster backwards ([8, 4096, 2048] bf16: 99 and
// 99, 140 and 158 us); with 128 tiles of 1024 tokens the chained form is faster ([4, 1024, 2048]: 16.6 -> 14.7, 23.5 -> 19.4 us and a
// clearing launch of 3), with 32 twice as fast (14.6 -> 9.0, 21 -> 10.3).
// Packed rows are as long as the table on the device says, so every tile has a workgroup there from 8192 tokens on: of [1, 65536, 2048]
// in 8 even rows the walk is 16 % faster (173 and 271 against 207 and 313 us), with all tokens in one of them four times as slow (811
// and 1258 against 206 and 312); of 512 rows the walk takes 342 and 583 us, the chained form 188 and 307.
// Of fewer than 8192 tokens no row is that long, and a clearing launch is what it would cost ([1, 5003, 1000] fp32 in 7 rows: 20.5 and
// 29.9 us walked, 21.2 and 29.8 chained, 6.6 to clear; so what bounds that batch is not its longest row).
bool chained(const lnx_linrec_args* a) {
  const int64_t wgs = (int64_t)rows_of(a) * channel_tiles(a);
  return a->T >= 8 * CTILE && (wgs < 160 || (a->nseq && a->T >= 64 * CTILE)) && slots_of(a, CTILE) * channel_tiles(a) <= MAX_GRID / CTHREADS;
}
// Bytes of what the workgroups leave for each other
int64_t pair_words(const lnx_linrec_args* a) { return 2 * (slots_of(a, CTILE) + slots_of(a, CTILE * GROUP)) * a->D; }
int64_t all_words(const lnx_linrec_args* a) { return pair_words(a) + (slots_of(a, CTILE * ANCHOR) * a->D + 3) / 4 * 4; }

int64_t token_stride(const lnx_linrec_args* a, int64_t stride) { return a->T > 1 ? stride : a->D; }

int check(const char* what, const lnx_linrec_args* a, bool bwd) {
  if (!a) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (a->B < 0 || a->T < 0 || a->D <= 0 || a->nseq < 0 || (a->nseq && a->B != 1))
    return lnx_set_error(LNX_ERR_SHAPE, "%s: unsupported dimensions B=%d T=%d D=%d nseq=%d", what, a->B, a->T, a->D, a->nseq);
  if ((a->dtype != LNX_F32 && a->dtype != LNX_BF16) || (a->g_dtype != LNX_F32 && a->g_dtype != a->dtype))
    return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d, g_dtype %d (x float32 or bfloat16, g float32 or x's type)", what, a->dtype, a->g_dtype);
  if (a->nseq && !a->cu_seqlens) return lnx_set_error(LNX_ERR_NULL, "%s: nseq without cu_seqlens", what);
  const bool tokens = (int64_t)a->B * a->T > 0, rows = rows_of(a) > 0;
  if (tokens && (!a->x || !a->g)) return lnx_set_error(LNX_ERR_NULL, "%s: x and g are required", what);
  if (!bwd && ((tokens && !a->y) || (rows && !a->final_state))) return lnx_set_error(LNX_ERR_NULL, "%s: y and final_state are required", what);
  if (bwd && tokens && (!a->d_x || !a->d_g || !a->kept)) return lnx_set_error(LNX_ERR_NULL, "%s: d_x, d_g and kept are required", what);
  // a lane's bytes within a tile are a 32-bit offset; the stride of a single token is never stepped over
  for (int64_t st : {token_stride(a, a->x_stride_t) * (a->dtype == LNX_BF16 ? 2 : 4), token_stride(a, a->g_stride_t) * (a->g_dtype == LNX_BF16 ? 2 : 4),
                     (bwd ? token_stride(a, a->d_y_stride_t) : 0) * (a->dtype == LNX_BF16 ? 2 : 4), (int64_t)a->D * 4})
    if (st < 0 || st > MAX_STRIDE) return lnx_set_error(LNX_ERR_SHAPE, "%s: tokens more than %lld bytes apart", what, (long long)MAX_STRIDE);
  if ((int64_t)rows_of(a) * channel_tiles(a) > MAX_GRID / THREADS) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  if (rows && chained(a)) {
    const uint64_t need = lnx_linrec_workspace_bytes(a);
    if (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16) return lnx_set_error(LNX_ERR_WORKSPACE, "%s: needs a workspace of %llu bytes", what, (unsigned long long)need);
  }
  return LNX_OK;
}

bool vectors(const void* p, int64_t sb, int64_t st, int64_t size) { return !p || (reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && sb % 4 == 0 && st % 4 == 0); }

Args kernel_args(const lnx_linrec_args* a) {
  Args k{};
  k.x = a->x, k.g = a->g, k.dy = a->d_y;
  k.xb = a->x_stride_b, k.gb = a->g_stride_b, k.yb = a->d_y_stride_b;
  k.xt = token_stride(a, a->x_stride_t), k.gt = token_stride(a, a->g_stride_t), k.yt = token_stride(a, a->d_y_stride_t);
  k.s0 = a->initial_state, k.ds = a->d_final_state, k.cu = a->cu_seqlens;
  k.y = a->y, k.dx = a->d_x, k.dg = a->d_g, k.sT = a->final_state, k.d0 = a->d_initial_state, k.kept = a->kept;
  k.T = a->T, k.D = a->D, k.ctiles = channel_tiles(a), k.packed = a->nseq != 0;
  if (chained(a)) {
    uint32_t* w = static_cast<uint32_t*>(a->workspace);
    k.pairs = reinterpret_cast<uint64_t*>(w), k.sums = k.pairs + slots_of(a, CTILE) * k.D, k.anchors = w + pair_words(a), k.counters = w + all_words(a);
  }
  return k;
}

template <typename T, typename G, bool VEC> void launch(const lnx_linrec_args* a, bool bwd, hipStream_t st) {
  const Args k = kernel_args(a);
  const int groups = (int)((int64_t)rows_of(a) * k.ctiles);
  if (chained(a)) {
    const int64_t words = all_words(a), threads = words / 4 + 1 > groups ? words / 4 + 1 : groups;
    lnx_profile_mark("linrec_clear", st);
    linrec_clear_kernel<<<dim3((unsigned)((threads + 255) / 256)), 256, 0, st>>>(static_cast<uint32_t*>(a->workspace), words, k.counters, groups);
    const dim3 grid((unsigned)(slots_of(a, CTILE) * k.ctiles));
    lnx_profile_mark(bwd ? "linrec_bwd_chain" : "linrec_fwd_chain", st);
    if (bwd) linrec_bwd_chain_kernel<T, G, VEC><<<grid, CTHREADS, 0, st>>>(k, rows_of(a));
    else linrec_fwd_chain_kernel<T, G, VEC><<<grid, CTHREADS, 0, st>>>(k, rows_of(a));
  } else {
    lnx_profile_mark(bwd ? "linrec_bwd" : "linrec_fwd", st);
    if (bwd) linrec_bwd_kernel<T, G, VEC><<<dim3((unsigned)groups), THREADS, 0, st>>>(k);
    else linrec_fwd_kernel<T, G, VEC><<<dim3((unsigned)groups), THREADS, 0, st>>>(k);
  }
}

int run(const char* what, const lnx_linrec_args* a, bool bwd, hipStream_t st) {
  if (int rc = check(what, a, bwd)) return rc;
  if (rows_of(a) == 0) return LNX_OK;
  const int64_t xs = a->dtype == LNX_BF16 ? 2 : 4, gs = a->g_dtype == LNX_BF16 ? 2 : 4;
  // four elements at a time: of the inputs with their strides, and of the outputs, whose rows are D long
  bool vec = a->D % 4 == 0 && vectors(a->x, a->x_stride_b, token_stride(a, a->x_stride_t), xs) && vectors(a->g, a->g_stride_b, token_stride(a, a->g_stride_t), gs) &&
             vectors(a->d_y, a->d_y_stride_b, token_stride(a, a->d_y_stride_t), xs);
  for (const void* p : {(const void*)a->y, (const void*)a->d_x}) vec = vec && reinterpret_cast<uintptr_t>(p) % (4 * xs) == 0;
  vec = vec && reinterpret_cast<uintptr_t>(a->d_g) % (4 * gs) == 0;
  if (a->dtype == LNX_F32) vec ? launch<float, float, true>(a, bwd, st) : launch<float, float, false>(a, bwd, st);
  else if (a->g_dtype == LNX_F32) vec ? launch<bf16_t, float, true>(a, bwd, st) : launch<bf16_t, float, false>(a, bwd, st);
  else vec ? launch<bf16_t, bf16_t, true>(a, bwd, st) : launch<bf16_t, bf16_t, false>(a, bwd, st);
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

template <typename T, typename G> void launch_step(const void* x, const void* g, const float* s, void* y, float* s_out, int64_t n, bool vec, hipStream_t st) {
  if (vec) linrec_step_kernel<T, G, 4><<<dim3((unsigned)((n / 4 + 255) / 256)), 256, 0, st>>>((const T*)x, (const G*)g, s, (T*)y, s_out, n);
  else linrec_step_kernel<T, G, 1><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>((const T*)x, (const G*)g, s, (T*)y, s_out, n);
}

}  // namespace

extern "C" uint64_t lnx_linrec_workspace_bytes(const lnx_linrec_args* a) {
  if (!a || a->D <= 0 || a->T < 0 || rows_of(a) <= 0) return 0;
  return chained(a) ? ((uint64_t)all_words(a) + (uint64_t)rows_of(a) * channel_tiles(a)) * sizeof(uint32_t) : 0;
}

extern "C" uint64_t lnx_linrec_kept_bytes(const lnx_linrec_args* a) {
  if (!a || a->D <= 0 || a->T < 0 || rows_of(a) <= 0) return 0;
  const uint64_t slots = a->nseq ? (uint64_t)a->T / KEPT + a->nseq : (uint64_t)a->B * (((int64_t)a->T + KEPT - 1) / KEPT);
  return slots * a->D * sizeof(float);
}

extern "C" int lnx_linrec_fwd(const lnx_linrec_args* a, void* hip_stream) { return run("linrec_fwd", a, false, static_cast<hipStream_t>(hip_stream)); }
extern "C" int lnx_linrec_bwd(const lnx_linrec_args* a, void* hip_stream) { return run("linrec_bwd", a, true, static_cast<hipStream_t>(hip_stream)); }

extern "C" int lnx_linrec_step(const void* x, const void* g, const float* state, void* y, float* new_state, int64_t n, int32_t dtype, int32_t g_dtype,
                               void* hip_stream) {
  if (n < 0 || n > (int64_t)1 << 38) return lnx_set_error(LNX_ERR_SHAPE, "linrec_step: n=%lld", (long long)n);
  if ((dtype != LNX_F32 && dtype != LNX_BF16) || (g_dtype != LNX_F32 && g_dtype != dtype))
    return lnx_set_error(LNX_ERR_DTYPE, "linrec_step: dtype %d, g_dtype %d", dtype, g_dtype);
  if (n == 0) return LNX_OK;
  if (!x || !g || !state || !y || !new_state) return lnx_set_error(LNX_ERR_NULL, "linrec_step: x, g, state, y and new_state are required");
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  bool vec = n % 4 == 0;
  for (const void* p : {x, g, (const void*)state, (const void*)y, (const void*)new_state}) vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  if ((vec ? n / 4 : n) > MAX_GRID - 256) return lnx_set_error(LNX_ERR_SHAPE, "linrec_step: n=%lld is too large for one launch", (long long)n);
  lnx_profile_mark("linrec_step", st);
  if (dtype == LNX_F32) launch_step<float, float>(x, g, state, y, new_state, n, vec, st);
  else if (g_dtype == LNX_F32) launch_step<bf16_t, float>(x, g, state, y, new_state, n, vec, st);
  else launch_step<bf16_t, bf16_t>(x, g, state, y, new_state, n, vec, st);
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "linrec_step: %s", hipGetErrorString(e));
}
