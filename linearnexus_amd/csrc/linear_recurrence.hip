// Element-wise gated linear recurrence over [rows, T, D] tensors, dense or packed, forward, backward and one token:
//   h_t = e^{g_t} h_{t-1} + x_t,  y_t = h_t                                    (h_0 the initial state, g log-decays)
//   dh_t = dy_t + e^{g_{t+1}} dh_{t+1},  dx_t = dh_t,  dg_t = e^{g_t} h_{t-1} dh_t,  dh_0 = e^{g_1} dh_1
// No products to speak of: every pass is bound by the bytes of its tensors.  A workgroup owns 128 bytes of channels of one row and
// walks its tokens in tiles of 256: a thread holds eight (bf16) or four (fp32) channels of four consecutive tokens as one 16-byte
// vector each and reduces them to a pair (A, H), the map h -> A h + H; pairs are scanned over the eight token groups of a wave by
// shuffles; the eight waves' pairs are chained through LDS by one lane per channel, which carries the state from tile to tile.  The
// loads of the next tile are in flight meanwhile.
// Everything between loads and stores is fp32.  The backward pass reads x again instead of y, which is rounded: the forward pass
// leaves the state entering every tile (fp32, 1 / 256 of x's elements), so the states behind dg are the unrounded ones.
// Where rows and channels give too few workgroups the tokens are cut into segments: a first launch reduces every segment to its
// pair, the second one starts each segment from the folded pairs before it.  No atomics: results are the same from run to run.
#include "lnx_common.h"
#include "mma_tiles.h"

namespace {

constexpr int THREADS = 512, WAVES = 8, TCOLS = 8, TROWS = THREADS / TCOLS;
constexpr int TILE = 4 * TROWS;  // tokens of a tile of the forward pass
// Tokens per thread of the backward pass, and so the distance of the states that the forward pass leaves for it: eight channels of
// four tokens would need 340 registers a lane.
template <typename T> constexpr int bwd_r() { return sizeof(T) == 2 ? 2 : 4; }
template <typename T> constexpr int kept_tokens() { return bwd_r<T>() * TROWS; }

// N consecutive elements as they lie in memory
template <typename E, int N> struct Raw {
  typedef typename Vec16<E>::V V;
  static constexpr int VN = Vec16<E>::N, K = N / VN;
  V v[K];
  template <bool VEC> __device__ __forceinline__ void load(const E* p, int left) {
    if (VEC) {
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = *reinterpret_cast<const V*>(p + k * VN);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i / VN][i % VN] = i < left ? p[i] : from_f32<E>(0.f);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = vec_zero<E>();
  }
  __device__ __forceinline__ float get(int i) const { return to_f32(v[i / VN][i % VN]); }
};

template <typename E, int N, bool VEC> __device__ __forceinline__ void put(E* p, const float (&f)[N], int left) {
  typedef typename Vec16<E>::V V;
  constexpr int VN = Vec16<E>::N;
#pragma unroll
  for (int k = 0; k < N / VN; ++k) {
    V v;
#pragma unroll
    for (int e = 0; e < VN; ++e) v[e] = from_f32<E>(f[k * VN + e]);
    if (VEC) *reinterpret_cast<V*>(p + k * VN) = v;
    else
#pragma unroll
      for (int e = 0; e < VN; ++e)
        if (k * VN + e < left) p[k * VN + e] = v[e];
  }
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

// What a workgroup works on: row, its first channel, its tiles
struct Place {
  int row, seg, len, ntile, per, tile0, tile1, c0, c, left;  // c0: the workgroup's first channel, c: this thread's
  int64_t tok, slot;  // first token in a packed batch (0 otherwise); first kept state
  __device__ __forceinline__ Place(const Args& a, int N, int TILE, int KEPT) {
    const int ct = blockIdx.x % a.ctiles, rs = blockIdx.x / a.ctiles;
    seg = rs % a.segs;
    row = rs / a.segs;
    if (a.packed) {
      const int first = seq_first(a.cu, row, a.T);
      len = seq_end(a.cu, row, a.T) - first;
      tok = first;
      slot = first / KEPT + row;
    } else {
      len = a.T;
      tok = 0;
      slot = (int64_t)row * ((a.T + KEPT - 1) / KEPT);
    }
    ntile = (len + TILE - 1) / TILE;
    per = (ntile + a.segs - 1) / a.segs;
    tile0 = min(seg * per, ntile);
    tile1 = min(tile0 + per, ntile);
    c0 = ct * TCOLS * N;
    c = c0 + (threadIdx.x & (TCOLS - 1)) * N;
    left = a.D - c;
  }
  template <typename E> __device__ __forceinline__ const E* at(const void* p, int64_t b, int64_t t, bool packed) const {
    return static_cast<const E*>(p) + (packed ? tok * t : row * b) + c;
  }
};

// Inclusive scan of the maps over the wave's eight token groups (lanes 8 apart), upwards or downwards in time
template <int N, bool UP> __device__ __forceinline__ void scan_wave(float (&A)[N], float (&H)[N], int lane) {
#pragma unroll
  for (int s = 8; s < 64; s <<= 1) {
    const bool on = UP ? lane >= s : lane < 64 - s;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float Ap = UP ? __shfl_up(A[i], s, LNX_WAVE) : __shfl_down(A[i], s, LNX_WAVE);
      const float Hp = UP ? __shfl_up(H[i], s, LNX_WAVE) : __shfl_down(H[i], s, LNX_WAVE);
      if (on) {
        H[i] += A[i] * Hp;
        A[i] *= Ap;
      }
    }
  }
}

// The eight waves' pairs and the states entering the waves, by channel of the workgroup
template <int N> struct Waves {
  static constexpr int C = TCOLS * N;
  float A[WAVES][C], H[WAVES][C], in[WAVES][C];
  // this wave's total out of its inclusive scan
  template <bool UP> __device__ __forceinline__ void leave(const float (&a)[N], const float (&h)[N], int lane, int wave) {
    if ((lane >> 3) == (UP ? 7 : 0)) {
      const int c = (lane & (TCOLS - 1)) * N;
#pragma unroll
      for (int i = 0; i < N; ++i) A[wave][c + i] = a[i], H[wave][c + i] = h[i];
    }
  }
  // one lane per channel: the state entering each wave, `carry` from before the tile to behind it; `all` the tile's product
  template <bool UP> __device__ __forceinline__ void chain(int c, float& carry, float& all) {
#pragma unroll
    for (int k = 0; k < WAVES; ++k) {
      const int w = UP ? k : WAVES - 1 - k;
      in[w][c] = carry;
      carry = A[w][c] * carry + H[w][c];
      all *= A[w][c];
    }
  }
  // the state entering this thread's tokens, from its wave's and the neighbouring groups' inclusive pairs
  template <bool UP> __device__ __forceinline__ void enter(const float (&a)[N], const float (&h)[N], float (&s)[N], int lane, int wave) const {
    const int c = (lane & (TCOLS - 1)) * N;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float Ap = UP ? __shfl_up(a[i], 8, LNX_WAVE) : __shfl_down(a[i], 8, LNX_WAVE);
      const float Hp = UP ? __shfl_up(h[i], 8, LNX_WAVE) : __shfl_down(h[i], 8, LNX_WAVE);
      const float from = in[wave][c + i];
      s[i] = (UP ? lane >= 8 : lane < 56) ? Ap * from + Hp : from;
    }
  }
};

// SUM: only the pair of each segment (but the last, which nothing follows)
template <typename T, typename G, bool VEC, bool SUM> __global__ __launch_bounds__(THREADS) void linrec_fwd_kernel(Args a) {
  constexpr int N = Vec16<T>::N, R = TILE / TROWS, KEPT = kept_tokens<T>(), C = TCOLS * N;
  __shared__ Waves<N> ws;
  const Place p(a, N, TILE, KEPT);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tr = threadIdx.x / TCOLS;
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
  const T* x = p.at<T>(a.x, a.xb, a.xt, a.packed);
  const G* g = p.at<G>(a.g, a.gb, a.gt, a.packed);
  T* y = static_cast<T*>(a.y) + (a.packed ? p.tok : (int64_t)p.row * a.T) * a.D + p.c;
  Raw<T, N> xr[R];
  Raw<G, N> gr[R];
  auto fetch = [&](int tile) {
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int64_t t = (int64_t)tile * TILE + tr * R + u;
      xr[u].zero();
      gr[u].zero();
      if (t < p.len && in_c) {
        xr[u].template load<VEC>(x + t * a.xt, p.left);
        gr[u].template load<VEC>(g + t * a.gt, p.left);
      }
    }
  };
  if (p.tile0 < p.tile1) fetch(p.tile0);
  for (int tile = p.tile0; tile < p.tile1; ++tile) {
    float e[R][N], xv[R][N], A[N], H[N];
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
    if (tile + 1 < p.tile1) fetch(tile + 1);
    scan_wave<N, true>(A, H, lane);
    ws.template leave<true>(A, H, lane, wave);
    lds_barrier();
    if (chains) {
      ws.template chain<true>(lane, carry, all);
      if (!SUM && a.kept && in_chan) {
#pragma unroll
        for (int k = 0; k < TILE / KEPT; ++k)
          if (tile * (int64_t)TILE + k * KEPT < p.len) a.kept[(p.slot + tile * (TILE / KEPT) + k) * a.D + chan] = ws.in[k * WAVES * KEPT / TILE][lane];
      }
    }
    lds_barrier();
    if (!SUM) {
      float h[N];
      ws.template enter<true>(A, H, h, lane, wave);
#pragma unroll
      for (int u = 0; u < R; ++u) {
        const int64_t t = (int64_t)tile * TILE + tr * R + u;
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = e[u][i] * h[i] + xv[u][i];
        if (t < p.len && in_c) put<T, N, VEC>(y + t * a.D, h, p.left);
      }
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
  constexpr int N = Vec16<T>::N, R = bwd_r<T>(), TILE = kept_tokens<T>(), C = TCOLS * N;
  __shared__ Waves<N> ws, wf;
  const Place p(a, N, TILE, TILE);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tr = threadIdx.x / TCOLS;
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
  const T* x = p.at<T>(a.x, a.xb, a.xt, a.packed);
  const G* g = p.at<G>(a.g, a.gb, a.gt, a.packed);
  const T* dy = p.at<T>(a.dy, a.yb, a.yt, a.packed);
  const int64_t base = (a.packed ? p.tok : (int64_t)p.row * a.T) * a.D + p.c;
  T* dx = static_cast<T*>(a.dx) + base;
  G* dg = static_cast<G*>(a.dg) + base;
  Raw<T, N> xr[R], yr[R];
  Raw<G, N> gr[R];
  auto fetch = [&](int tile) {
    if (states && chan < a.D) start = a.kept[(p.slot + tile) * a.D + chan];
#pragma unroll
    for (int u = 0; u < R; ++u) {
      const int64_t t = (int64_t)tile * TILE + tr * R + u;
      xr[u].zero();
      yr[u].zero();
      gr[u].zero();
      if (t < p.len && in_c) {
        if (!SUM) xr[u].template load<VEC>(x + t * a.xt, p.left);
        if (a.dy) yr[u].template load<VEC>(dy + t * a.yt, p.left);
        gr[u].template load<VEC>(g + t * a.gt, p.left);
      }
    }
  };
  if (p.tile0 < p.tile1) fetch(p.tile1 - 1);
  for (int tile = p.tile1 - 1; tile >= p.tile0; --tile) {
    float e[R][N], xv[R][N], dyv[R][N], A[N], H[N], Af[N], Hf[N];
#pragma unroll
    for (int i = 0; i < N; ++i) A[i] = 1.f, H[i] = 0.f, Hf[i] = 0.f;
#pragma unroll
    for (int u = R - 1; u >= 0; --u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        e[u][i] = __expf(gr[u].get(i));
        dyv[u][i] = yr[u].get(i);
        H[i] = e[u][i] * (dyv[u][i] + H[i]);
        A[i] *= e[u][i];
      }
    if (!SUM) {
#pragma unroll
      for (int u = 0; u < R; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) xv[u][i] = xr[u].get(i), Hf[i] = e[u][i] * Hf[i] + xv[u][i];
    }
    float from = start;
    if (tile > p.tile0) fetch(tile - 1);
    if (!SUM) {
#pragma unroll
      for (int i = 0; i < N; ++i) Af[i] = A[i];
      scan_wave<N, true>(Af, Hf, lane);
      wf.template leave<true>(Af, Hf, lane, wave);
    }
    scan_wave<N, false>(A, H, lane);
    ws.template leave<false>(A, H, lane, wave);
    lds_barrier();
    if (chains) ws.template chain<false>(lane, carry, all);
    if (states) {
      float none = 1.f;
      wf.template chain<true>(lane, from, none);
    }
    lds_barrier();
    if (!SUM) {
      float h[N], o[N], hb[R][N];
      wf.template enter<true>(Af, Hf, h, lane, wave);
      ws.template enter<false>(A, H, o, lane, wave);
#pragma unroll
      for (int u = 0; u < R; ++u)
#pragma unroll
        for (int i = 0; i < N; ++i) hb[u][i] = h[i], h[i] = e[u][i] * h[i] + xv[u][i];
#pragma unroll
      for (int u = R - 1; u >= 0; --u) {
        const int64_t t = (int64_t)tile * TILE + tr * R + u;
        float dh[N], dgv[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          dh[i] = dyv[u][i] + o[i];
          o[i] = e[u][i] * dh[i];
          dgv[i] = hb[u][i] * o[i];
        }
        if (t < p.len && in_c) {
          put<T, N, VEC>(dx + t * a.D, dh, p.left);
          put<G, N, VEC>(dg + t * a.D, dgv, p.left);
        }
      }
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
template <typename T, typename G, int N> __global__ __launch_bounds__(256) void linrec_step_kernel(const T* x, const G* g, const float* s, T* y, float* s_out, int64_t n) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * N;
  if (i >= n) return;
  if (N == 4) {
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

int rows_of(const lnx_linrec_args* a) { return a->nseq ? a->nseq : a->B; }
int channel_tiles(const lnx_linrec_args* a) {
  const int w = TCOLS * (a->dtype == LNX_BF16 ? 8 : 4);
  return (a->D + w - 1) / w;
}

// Segments of a row's tokens: as many as bring the launch to one workgroup a CU, of four tiles each at least (the first launch
// reads the inputs once more, so a launch that fills the chip by itself is not cut).
int segments(const lnx_linrec_args* a) {
  const int64_t wgs = (int64_t)rows_of(a) * channel_tiles(a), tiles = (a->T + TILE - 1) / TILE;
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
  if ((int64_t)rows_of(a) * channel_tiles(a) * segments(a) > 0x7fffffff) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  if (rows && segments(a) > 1) {
    const uint64_t need = lnx_linrec_workspace_bytes(a);
    if (!a->workspace || a->workspace_bytes < need) return lnx_set_error(LNX_ERR_WORKSPACE, "%s: needs a workspace of %llu bytes", what, (unsigned long long)need);
  }
  return LNX_OK;
}

bool vectors(const void* p, int64_t sb, int64_t st, int64_t size) { return !p || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && sb * size % 16 == 0 && st * size % 16 == 0); }

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
  // rows as 16-byte vectors: of the inputs with their strides, and of everything that is [.., D] itself
  bool vec = a->D * xs % 16 == 0 && vectors(a->x, a->x_stride_b, a->x_stride_t, xs) && vectors(a->g, a->g_stride_b, a->g_stride_t, gs) &&
             vectors(a->d_y, a->d_y_stride_b, a->d_y_stride_t, xs);
  for (const void* p : {(const void*)a->initial_state, (const void*)a->y, (const void*)a->final_state, (const void*)a->kept, (const void*)a->workspace,
                        (const void*)a->d_final_state, (const void*)a->d_x, (const void*)a->d_g, (const void*)a->d_initial_state})
    vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
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
  const int kept = a->dtype == LNX_BF16 ? kept_tokens<bf16_t>() : kept_tokens<float>();
  const uint64_t slots = a->nseq ? (uint64_t)a->T / kept + a->nseq : (uint64_t)a->B * ((a->T + kept - 1) / kept);
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
