// Element-wise gated linear recurrence over [rows, T, D] tensors, dense or packed, forward, backward and one token:
//   h_t = e^{g_t} h_{t-1} + x_t,  y_t = h_t                                    (h_0 the initial state, g log-decays)
//   dh_t = dy_t + e^{g_{t+1}} dh_{t+1},  dx_t = dh_t,  dg_t = e^{g_t} h_{t-1} dh_t,  dh_0 = e^{g_1} dh_1
// No products to speak of: every pass is bound by the bytes of its tensors.  A workgroup owns 128 bytes of channels of one row and walks
// its tokens in tiles: a thread holds four channels of R consecutive tokens and reduces them to a pair (A, H), the map h -> A h + H;
// pairs are scanned over the token groups of a wave by lane swaps, and the eight waves' pairs are chained through LDS by one lane per
// channel, which carries the state from tile to tile.  The loads of the next tile are in flight meanwhile.  (Eight channels of four
// tokens a thread, scanned over eight groups by shuffles, were bound by the scan: 4.1 TB/s at [8, 4096, 2048] bf16, the same with
// twice the loads in flight.)  Everything between loads and stores is fp32.  The backward pass reads x again instead of y, which is
// rounded: the forward pass leaves the state entering every tile (fp32, 1 / 256 of the elements), so the states
// behind dg are the unrounded ones.
// Where rows and channels give too few workgroups the tokens are cut into segments: a first launch reduces every segment to its
// pair, the second one starts each segment from the folded pairs before it.  No atomics: results are the same from run to run.
#include "lnx_common.h"
#include "mma_tiles.h"

namespace {

constexpr int THREADS = 512, WAVES = 8, N = 4, TILE = 256;  // tokens of a tile
// By element type: threads side by side in a row, so that a row of a workgroup is 128 bytes; its channels; tokens per thread (what the
// backward pass's registers take)
template <typename T> struct Shape {
  static constexpr int COLS = sizeof(T) == 2 ? 16 : 8, C = COLS * N, R = TILE * COLS / THREADS;
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
  float *sT, *d0, *kept, *pairs;
  int T, D, ctiles, segs;
  bool packed;
};

// What a workgroup works on: row, its channels, its tiles
template <typename T> struct Place {
  int row, seg, len, ntile, per, tile0, tile1, c0, c, left;  // c0: the workgroup's first channel, c: this thread's
  int64_t tok, slot;  // first token in a packed batch (0 otherwise); first kept state
  __device__ __forceinline__ Place(const Args& a) {
    const int ct = blockIdx.x % a.ctiles, rs = blockIdx.x / a.ctiles;
    seg = rs % a.segs;
    row = rs / a.segs;
    if (a.packed) {
      const int first = seq_first(a.cu, row, a.T);
      len = seq_end(a.cu, row, a.T) - first;
      tok = first;
      slot = first / TILE + row;
    } else {
      len = a.T;
      tok = 0;
      slot = (int64_t)row * ((a.T + TILE - 1) / TILE);
    }
    ntile = (len + TILE - 1) / TILE;
    per = (ntile + a.segs - 1) / a.segs;
    tile0 = min(seg * per, ntile);
    tile1 = min(tile0 + per, ntile);
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

// The eight waves' pairs and the states entering the waves, by channel of the workgroup
template <int COLS> struct Waves {
  static constexpr int C = COLS * N;
  float A[WAVES][C], H[WAVES][C], in[WAVES][C];
  __device__ __forceinline__ void leave(const float (&a)[N], const float (&h)[N], int lane, int wave) {
    if (lane < COLS) {
      store4(&A[wave][lane * N], floatx4{a[0], a[1], a[2], a[3]});
      store4(&H[wave][lane * N], floatx4{h[0], h[1], h[2], h[3]});
    }
  }
  // one lane per channel: the state entering each wave, `carry` from before the tile to behind it; `all` the tiles' product
  template <bool UP> __device__ __forceinline__ void chain(int c, float& carry, float& all) {
    float a[WAVES], h[WAVES];
#pragma unroll
    for (int w = 0; w < WAVES; ++w) a[w] = A[w][c], h[w] = H[w][c];
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const int w = UP ? k : WAVES - 1 - k;
      in[w][c] = carry;
      carry = a[w] * carry + h[w];
      all *= a[w];
    }
  }
  // the state entering this thread's tokens
  __device__ __forceinline__ void enter(const float (&ea)[N], const float (&eh)[N], float (&s)[N], int lane, int wave) const {
    const floatx4 from = load4(&in[wave][(lane & (COLS - 1)) * N]);
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = ea[i] * from[i] + eh[i];
  }
};

// SUM: only the pair of each segment (but the last, which nothing follows)
template <typename T, typename G, bool VEC, bool SUM> __global__ __launch_bounds__(THREADS) void linrec_fwd_kernel(Args a) {
  constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  __shared__ Waves<COLS> ws;
  const Place<T> p(a);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tr = threadIdx.x / COLS;
  if (SUM && p.tile1 >= p.ntile) return;
  const bool in_c = p.left > 0;
  // the chain's lanes: one channel each
  const int chan = p.c0 + lane;
  const bool chains = wave == 0 && lane < C, in_chan = chains && chan < a.D;
  const int64_t row_c = (int64_t)p.row * a.D + chan;
  float carry = 0.f, all = 1.f;
  if (!SUM && in_chan) {
    if (a.s0) carry = a.s0[row_c];
    if (p.tile0 < p.tile1)
      for (int s = 0; s < p.seg; ++s) {
        const float* q = a.pairs + ((int64_t)p.row * a.segs + s) * 2 * a.D + chan;
        carry = q[0] * carry + q[a.D];
      }
  }
  const int64_t first = (int64_t)p.tile0 * TILE, row_b = a.packed ? 0 : 1;  // a packed batch is one row
  const char* x = p.template at<T>(a.x, row_b * a.xb, a.xt, first);
  const char* g = p.template at<G>(a.g, row_b * a.gb, a.gt, first);
  char* y = const_cast<char*>(p.template at<T>(a.y, row_b * a.T * a.D, a.D, first));
  const unsigned xo = p.template lane<T>(a.xt, tr * R), go = p.template lane<G>(a.gt, tr * R), yo = p.template lane<T>(a.D, tr * R);
  const int64_t xs = a.xt * (int64_t)sizeof(T), gs = a.gt * (int64_t)sizeof(G), ys = a.D * (int64_t)sizeof(T);
  Raw<T, VEC> xr[R];
  Raw<G, VEC> gr[R];
  // the tile that x and g point at
  const auto fetch = [&](int tile) {
    if ((tile + 1) * (int64_t)TILE <= p.len && p.c0 + C <= a.D) {
#pragma unroll
      for (int u = 0; u < R; ++u) xr[u].load(elems<T>(x + u * xs, xo), N), gr[u].load(elems<G>(g + u * gs, go), N);
    } else {
#pragma unroll
      for (int u = 0; u < R; ++u) {
        xr[u].zero();
        gr[u].zero();
        if ((int64_t)tile * TILE + tr * R + u < p.len && in_c) xr[u].load(elems<T>(x + u * xs, xo), p.left), gr[u].load(elems<G>(g + u * gs, go), p.left);
      }
    }
  };
  if (p.tile0 < p.tile1) fetch(p.tile0);
  for (int tile = p.tile0; tile < p.tile1; ++tile) {
    float e[R][N], xv[R][N], A[N], H[N], ea[N], eh[N];
#pragma unroll
    for (int i = 0; i < N; ++i) A[i] = 1.f, H[i] = 0.f;
#pragma unroll
    for (int u = 0; u < R; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        e[u][i] = __expf(gr[u].get(i));  // 1 behind the end: the state stands
        xv[u][i] = xr[u].get(i);
        H[i] = e[u][i] * H[i] + xv[u][i];
        A[i] *= e[u][i];
      }
    x += TILE * xs;
    g += TILE * gs;
    if (tile + 1 < p.tile1) fetch(tile + 1);
#pragma unroll
    for (int i = 0; i < N; ++i) scan_wave<COLS, true>(A[i], H[i], ea[i], eh[i], lane);
    ws.leave(A, H, lane, wave);
    lds_barrier();
    if (chains) {
      if (!SUM && a.kept && in_chan) a.kept[(p.slot + tile) * a.D + chan] = carry;
      ws.template chain<true>(lane, carry, all);
    }
    lds_barrier();
    if (!SUM) {
      float h[N];
      ws.enter(ea, eh, h, lane, wave);
      const bool whole = (tile + 1) * (int64_t)TILE <= p.len && p.c0 + C <= a.D;
#pragma unroll
      for (int u = 0; u < R; ++u) {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = e[u][i] * h[i] + xv[u][i];
        if (whole || ((int64_t)tile * TILE + tr * R + u < p.len && in_c)) put<VEC>(elems<T>(y + u * ys, yo), h, p.left);
      }
      y += TILE * ys;
    }
  }
  if (!in_chan) return;
  if (SUM) {
    float* q = a.pairs + ((int64_t)p.row * a.segs + p.seg) * 2 * a.D + chan;
    q[0] = all;
    q[a.D] = carry;
  } else if (p.ntile ? p.tile0 < p.tile1 && p.tile1 == p.ntile : p.seg == 0) {
    a.sT[row_c] = carry;
  }
}

// Backwards in time: o is e^{g_{t+1}} dh_{t+1}.  SUM: only the pair of each segment (but the first, which nothing precedes)
template <typename T, typename G, bool VEC, bool SUM> __global__ __launch_bounds__(THREADS) void linrec_bwd_kernel(Args a) {
  constexpr int R = Shape<T>::R, COLS = Shape<T>::COLS, C = Shape<T>::C;
  __shared__ Waves<COLS> ws, wf;
  const Place<T> p(a);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tr = threadIdx.x / COLS;
  if (SUM && (p.seg == 0 || p.tile0 >= p.tile1)) return;
  const bool in_c = p.left > 0;
  const int chan = p.c0 + lane;  // wave 0 chains the gradients, wave 1 the states
  const bool chains = wave == 0 && lane < C, in_chan = chains && chan < a.D, states = !SUM && wave == 1 && lane < C;
  const int64_t row_c = (int64_t)p.row * a.D + chan;
  float carry = 0.f, all = 1.f, start = 0.f;
  if (!SUM && in_chan) {
    if (a.ds) carry = a.ds[row_c];
    if (p.tile0 < p.tile1)
      for (int s = (p.ntile - 1) / p.per; s > p.seg; --s) {
        const float* q = a.pairs + ((int64_t)p.row * a.segs + s) * 2 * a.D + chan;
        carry = q[0] * carry + q[a.D];
      }
  }
  const int64_t first = (int64_t)(p.tile1 - 1) * TILE, row_b = a.packed ? 0 : 1;  // of the last tile
  const char* x = p.template at<T>(a.x, row_b * a.xb, a.xt, first);
  const char* g = p.template at<G>(a.g, row_b * a.gb, a.gt, first);
  const char* dy = p.template at<T>(a.dy, row_b * a.yb, a.yt, first);
  char* dx = const_cast<char*>(p.template at<T>(a.dx, row_b * a.T * a.D, a.D, first));
  char* dg = const_cast<char*>(p.template at<G>(a.dg, row_b * a.T * a.D, a.D, first));
  const unsigned xo = p.template lane<T>(a.xt, tr * R), go = p.template lane<G>(a.gt, tr * R), yo = p.template lane<T>(a.yt, tr * R), dxo = p.template lane<T>(a.D, tr * R), dgo = p.template lane<G>(a.D, tr * R);
  const int64_t xs = a.xt * (int64_t)sizeof(T), gs = a.gt * (int64_t)sizeof(G), ys = a.yt * (int64_t)sizeof(T), dxs = a.D * (int64_t)sizeof(T), dgs = a.D * (int64_t)sizeof(G);
  Raw<T, VEC> xr[R], yr[R];
  Raw<G, VEC> gr[R];
  if (!a.dy)
#pragma unroll
    for (int u = 0; u < R; ++u) yr[u].zero();
  const auto fetch = [&](int tile) {
    if (states && chan < a.D) start = a.kept[(p.slot + tile) * a.D + chan];
    if ((tile + 1) * (int64_t)TILE <= p.len && p.c0 + C <= a.D) {
#pragma unroll
      for (int u = 0; u < R; ++u) {
        if (!SUM) xr[u].load(elems<T>(x + u * xs, xo), N);
        gr[u].load(elems<G>(g + u * gs, go), N);
      }
      if (a.dy)
#pragma unroll
        for (int u = 0; u < R; ++u) yr[u].load(elems<T>(dy + u * ys, yo), N);
    } else {
#pragma unroll
      for (int u = 0; u < R; ++u) {
        xr[u].zero();
        yr[u].zero();
        gr[u].zero();
        if ((int64_t)tile * TILE + tr * R + u < p.len && in_c) {
          if (!SUM) xr[u].load(elems<T>(x + u * xs, xo), p.left);
          if (a.dy) yr[u].load(elems<T>(dy + u * ys, yo), p.left);
          gr[u].load(elems<G>(g + u * gs, go), p.left);
        }
      }
    }
  };
  if (p.tile0 < p.tile1) fetch(p.tile1 - 1);
  for (int tile = p.tile1 - 1; tile >= p.tile0; --tile) {
    float e[R][N], A[N], H[N], ea[N], eh[N], Af[N], Hf[N], fa[N], fh[N];
    Raw<T, VEC> xk[R], yk[R];
#pragma unroll
    for (int i = 0; i < N; ++i) A[i] = 1.f, H[i] = 0.f, Hf[i] = 0.f;
#pragma unroll
    for (int u = R - 1; u >= 0; --u) {
      xk[u] = xr[u];
      yk[u] = yr[u];
#pragma unroll
      for (int i = 0; i < N; ++i) {
        e[u][i] = __expf(gr[u].get(i));
        H[i] = e[u][i] * (yk[u].get(i) + H[i]);
        A[i] *= e[u][i];
      }
    }
    if (!SUM)
#pragma unroll
      for (int u = 0; u < R; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) Hf[i] = e[u][i] * Hf[i] + xk[u].get(i);
    float from = start;
    x -= TILE * xs;
    g -= TILE * gs;
    dy -= TILE * ys;
    if (tile > p.tile0) fetch(tile - 1);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (!SUM) {
        Af[i] = A[i];
        scan_wave<COLS, true>(Af[i], Hf[i], fa[i], fh[i], lane);
      }
      scan_wave<COLS, false>(A[i], H[i], ea[i], eh[i], lane);
    }
    if (!SUM) wf.leave(Af, Hf, lane, wave);
    ws.leave(A, H, lane, wave);
    lds_barrier();
    if (chains) ws.template chain<false>(lane, carry, all);
    if (states) {
      float none = 1.f;
      wf.template chain<true>(lane, from, none);
    }
    lds_barrier();
    if (!SUM) {
      float h[N], o[N], hb[R][N];
      wf.enter(fa, fh, h, lane, wave);
      ws.enter(ea, eh, o, lane, wave);
      const bool whole = (tile + 1) * (int64_t)TILE <= p.len && p.c0 + C <= a.D;
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
        if (whole || ((int64_t)tile * TILE + tr * R + u < p.len && in_c)) {
          put<VEC>(elems<T>(dx + u * dxs, dxo), dh, p.left);
          put<VEC>(elems<G>(dg + u * dgs, dgo), dgv, p.left);
        }
      }
      dx -= TILE * dxs;
      dg -= TILE * dgs;
    }
  }
  if (!in_chan) return;
  if (SUM) {
    float* q = a.pairs + ((int64_t)p.row * a.segs + p.seg) * 2 * a.D + chan;
    q[0] = all;
    q[a.D] = carry;
  } else if (a.d0 && p.seg == 0) {
    a.d0[row_c] = carry;
  }
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

constexpr int64_t MAX_STRIDE = 4 << 20;
int rows_of(const lnx_linrec_args* a) { return a->nseq ? a->nseq : a->B; }
int channel_tiles(const lnx_linrec_args* a) {
  const int c = a->dtype == LNX_BF16 ? Shape<bf16_t>::C : Shape<float>::C;
  return (int)(((int64_t)a->D + c - 1) / c);
}

// Segments of a row's tokens: as many as bring the launch to one workgroup a CU, of four tiles each at least (the first launch
// reads the inputs once more, so a launch that nearly fills the chip by itself is not cut).
int segments(const lnx_linrec_args* a) {
  const int64_t wgs = (int64_t)rows_of(a) * channel_tiles(a), len = a->nseq ? a->T / a->nseq : a->T, tiles = (len + TILE - 1) / TILE;  // of the average sequence
  int64_t s = wgs >= 160 ? 1 : 256 / (wgs > 0 ? wgs : 1);
  if (s > tiles / 4) s = tiles / 4;
  return s < 1 ? 1 : (int)s;
}

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
  // a lane's bytes within a tile are a 32-bit offset
  for (int64_t st : {a->x_stride_t * (a->dtype == LNX_BF16 ? 2 : 4), a->g_stride_t * (a->g_dtype == LNX_BF16 ? 2 : 4), (bwd ? a->d_y_stride_t : 0) * (a->dtype == LNX_BF16 ? 2 : 4),
                     (int64_t)a->D * 4})
    if (st < 0 || st > MAX_STRIDE) return lnx_set_error(LNX_ERR_SHAPE, "%s: tokens more than %lld bytes apart", what, (long long)MAX_STRIDE);
  if ((int64_t)rows_of(a) * channel_tiles(a) * segments(a) > 0x7fffffff) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  if (rows && segments(a) > 1) {
    const uint64_t need = lnx_linrec_workspace_bytes(a);
    if (!a->workspace || a->workspace_bytes < need) return lnx_set_error(LNX_ERR_WORKSPACE, "%s: needs a workspace of %llu bytes", what, (unsigned long long)need);
  }
  return LNX_OK;
}

bool vectors(const void* p, int64_t sb, int64_t st, int64_t size) { return !p || (reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && sb % 4 == 0 && st % 4 == 0); }

Args kernel_args(const lnx_linrec_args* a, int segs) {
  Args k{};
  k.x = a->x, k.g = a->g, k.dy = a->d_y;
  k.xb = a->x_stride_b, k.xt = a->x_stride_t, k.gb = a->g_stride_b, k.gt = a->g_stride_t, k.yb = a->d_y_stride_b, k.yt = a->d_y_stride_t;
  k.s0 = a->initial_state, k.ds = a->d_final_state, k.cu = a->cu_seqlens;
  k.y = a->y, k.dx = a->d_x, k.dg = a->d_g, k.sT = a->final_state, k.d0 = a->d_initial_state, k.kept = a->kept;
  k.pairs = static_cast<float*>(a->workspace);
  k.T = a->T, k.D = a->D, k.ctiles = channel_tiles(a), k.segs = segs, k.packed = a->nseq != 0;
  return k;
}

template <typename T, typename G, bool VEC> void launch(const lnx_linrec_args* a, bool bwd, hipStream_t st) {
  const int segs = segments(a);
  const Args k = kernel_args(a, segs);
  const dim3 grid((unsigned)((int64_t)rows_of(a) * k.ctiles * segs));
  if (bwd) {
    if (segs > 1) {
      lnx_profile_mark("linrec_bwd_pairs", st);
      linrec_bwd_kernel<T, G, VEC, true><<<grid, THREADS, 0, st>>>(k);
    }
    lnx_profile_mark("linrec_bwd", st);
    linrec_bwd_kernel<T, G, VEC, false><<<grid, THREADS, 0, st>>>(k);
  } else {
    if (segs > 1) {
      lnx_profile_mark("linrec_fwd_pairs", st);
      linrec_fwd_kernel<T, G, VEC, true><<<grid, THREADS, 0, st>>>(k);
    }
    lnx_profile_mark("linrec_fwd", st);
    linrec_fwd_kernel<T, G, VEC, false><<<grid, THREADS, 0, st>>>(k);
  }
}

int run(const char* what, const lnx_linrec_args* a, bool bwd, hipStream_t st) {
  if (int rc = check(what, a, bwd)) return rc;
  if (rows_of(a) == 0) return LNX_OK;
  const int64_t xs = a->dtype == LNX_BF16 ? 2 : 4, gs = a->g_dtype == LNX_BF16 ? 2 : 4;
  // four elements at a time: of the inputs with their strides, and of the outputs, whose rows are D long
  bool vec = a->D % 4 == 0 && vectors(a->x, a->x_stride_b, a->x_stride_t, xs) && vectors(a->g, a->g_stride_b, a->g_stride_t, gs) &&
             vectors(a->d_y, a->d_y_stride_b, a->d_y_stride_t, xs);
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
  const int s = segments(a);
  return s > 1 ? (uint64_t)rows_of(a) * s * 2 * a->D * sizeof(float) : 0;
}

extern "C" uint64_t lnx_linrec_kept_bytes(const lnx_linrec_args* a) {
  if (!a || a->D <= 0 || a->T < 0 || rows_of(a) <= 0) return 0;
  const uint64_t slots = a->nseq ? (uint64_t)a->T / TILE + a->nseq : (uint64_t)a->B * (((int64_t)a->T + TILE - 1) / TILE);
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
  lnx_profile_mark("linrec_step", st);
  if (dtype == LNX_F32) launch_step<float, float>(x, g, state, y, new_state, n, vec, st);
  else if (g_dtype == LNX_F32) launch_step<bf16_t, float>(x, g, state, y, new_state, n, vec, st);
  else launch_step<bf16_t, bf16_t>(x, g, state, y, new_state, n, vec, st);
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "linrec_step: %s", hipGetErrorString(e));
}
