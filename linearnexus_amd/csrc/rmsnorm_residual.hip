// The norms around a block on its residual stream, one pass over the rows forward and one backward:
//   u = [RMSNorm(x) * post] * [sigmoid(gate)]     r' = r + scale * u     z = RMSNorm(r') * weight
// (bracketed factors and r are optional; scale is a number or one factor per column).  With xn = x rho (x without the norm), s the
// sigmoid, c the scale, D the whole gradient of r':
//   D = dr' + rho2 (dz w - r' rho2^2 mean(dz w r'))        dr = D          dw = sum dz r' rho2
//   v = D c post s      dx = rho (v - x rho^2 mean(v x))   dgate = D c post xn s (1 - s)
//   S = sum D s xn      dpost = c S                        dscale = post S
// Bound by bytes: a row (or several) belongs to one workgroup, is read once with 16-byte loads and stays in registers between its
// two reductions.  The backward pass forms r' again from its inputs in fp32 instead of reading the rounded one: the same bytes, and
// no rounding of the stream enters the sums over the rows, which are fp32 outputs.  Those sums stay in registers over all rows of a
// workgroup and leave as one partial row each; a second launch adds them (no atomics, the same from run to run).
// 32768 rows of 2048, bf16 with an fp32 stream and all options: forward 160-170 us for 940 MB (5.5-5.9 TB/s), backward 281-289 for 1.48 GB
// (5.1-5.3 TB/s) and 8 for the sums; a copy reaches 4.97.  16384 rows of 2048 in fp32: 126 and 207 us (5.3 and 5.2 TB/s).  Of 4097 to 8192 fp32
// columns the backward pass spills some 40 registers: 4096 rows of 8192 take 294 us, 8192 of 4096 208.
#include "lnx_common.h"
#include "mma_tiles.h"
#include "reduce_rows.h"
#include "row_vectors.h"

namespace {

__device__ __forceinline__ float sigmoid(float z) { return 1.f / (1.f + __expf(-z)); }

struct Args {
  const void *x, *r, *gate;
  const float *w, *post, *scale_v;
  void *z, *out;
  const void *dz, *dout;
  void *dx, *dr, *dgate;
  float* dw;  // partial rows
  int64_t rows;
  int d, dpad;
  float scale, eps, inv_d;
};

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

template <typename T, typename S, typename G, int TPR, int K, bool VEC> __global__ __launch_bounds__(block_of(TPR)) void rmsnorm_residual_fwd_kernel(Args a) {
  constexpr int VN = Vec16<T>::N, RPB = block_of(TPR) / TPR, ES = VEC ? 1 : TPR;
  __shared__ float red[2][16];
  const int li = threadIdx.x % TPR;
  const int64_t row = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * RPB + threadIdx.x / TPR;
  if (row >= a.rows) return;  // whole waves: rows of one wave have no barrier
  const int64_t base = row * a.d;
  const T* x = static_cast<const T*>(a.x) + base;
  const G* gate = a.gate ? static_cast<const G*>(a.gate) + base : nullptr;
  const S* r = a.r ? static_cast<const S*>(a.r) + base : nullptr;
  float xv[K][VN], rv[K][VN], gv[K][VN], ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = first_column<TPR, VN, ES>(k, li), left = a.d - c;
#pragma unroll
    for (int e = 0; e < VN; ++e) xv[k][e] = rv[k][e] = gv[k][e] = 0.f;
    if (left > 0) {
      load_row<T, VN, ES>(x + c, left, xv[k]);
      if (r) load_row<S, VN, ES>(r + c, left, rv[k]);
      if (gate) load_row<G, VN, ES>(gate + c, left, gv[k]);
    }
  }
  float rho = 1.f;
  if (a.post) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) ss += xv[k][e] * xv[k][e];
    rho = rsqrtf(row_sum<TPR>(ss, red[0]) * a.inv_d + a.eps);
  }
  ss = 0.f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = first_column<TPR, VN, ES>(k, li), left = a.d - c;
    if (left > 0) {
      float pv[VN], sv[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) pv[e] = 1.f, sv[e] = a.scale;
      if (a.post) load_row<float, VN, ES>(a.post + c, left, pv);
      if (a.scale_v) load_row<float, VN, ES>(a.scale_v + c, left, sv);
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        float u = xv[k][e] * rho * (pv[e] * sv[e]);
        if (gate) u *= sigmoid(gv[k][e]);
        rv[k][e] += u;
        ss += rv[k][e] * rv[k][e];
      }
      if (a.out) store_row<S, VN, ES>(static_cast<S*>(a.out) + base + c, left, rv[k]);
    }
  }
  if (!a.z) return;
  const float rho2 = rsqrtf(row_sum<TPR>(ss, red[1]) * a.inv_d + a.eps);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = first_column<TPR, VN, ES>(k, li), left = a.d - c;
    if (left > 0) {
      float wv[VN], zv[VN];
      load_row<float, VN, ES>(a.w + c, left, wv);
#pragma unroll
      for (int e = 0; e < VN; ++e) zv[e] = rv[k][e] * rho2 * wv[e];
      store_row<T, VN, ES>(static_cast<T*>(a.z) + base + c, left, zv);
    }
  }
}

// Rows blockIdx, blockIdx + gridDim, ...; the next row is on its way while one is worked on.
template <typename T, typename S, typename G, int TPR, int K, bool VEC> __global__ __launch_bounds__(block_of(TPR)) void rmsnorm_residual_bwd_kernel(Args a) {
  constexpr int VN = Vec16<T>::N, RPB = block_of(TPR) / TPR, C = TPR * K * VN, ES = VEC ? 1 : TPR;
  __shared__ float red[2][3][32];
  const int li = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  float wv[K][VN], cp[K][VN], dw[K][VN], db[K][VN];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = first_column<TPR, VN, ES>(k, li), left = a.d - c;
#pragma unroll
    for (int e = 0; e < VN; ++e) wv[k][e] = dw[k][e] = db[k][e] = 0.f, cp[k][e] = a.scale;
    if (left > 0) {
      float t[VN];
      if (a.w) load_row<float, VN, ES>(a.w + c, left, wv[k]);
      if (a.scale_v) load_row<float, VN, ES>(a.scale_v + c, left, cp[k]);
      if (a.post) {
        load_row<float, VN, ES>(a.post + c, left, t);
#pragma unroll
        for (int e = 0; e < VN; ++e) cp[k][e] *= t[e];
      }
    }
  }
  RawRow<T, VN, ES> xr[K], zr[K];
  RawRow<G, VN, ES> gr[K];
  RawRow<S, VN, ES> rr[K], orr[K];
  auto fetch = [&](int64_t row) {
    const int64_t base = row * a.d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = first_column<TPR, VN, ES>(k, li), left = row < a.rows ? a.d - c : 0;
      const int64_t at = base + c;
      xr[k].load(static_cast<const T*>(a.x) + at, left);
      if (a.r) rr[k].load(static_cast<const S*>(a.r) + at, left);
      else rr[k].zero();
      if (a.gate) gr[k].load(static_cast<const G*>(a.gate) + at, left);
      else gr[k].zero();
      if (a.dz) zr[k].load(static_cast<const T*>(a.dz) + at, left);
      else zr[k].zero();
      if (a.dout) orr[k].load(static_cast<const S*>(a.dout) + at, left);
      else orr[k].zero();
    }
  };
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)blockIdx.x * RPB + sub;
  fetch(row);
  // every thread of a workgroup of one row takes the same number of turns (barriers); waves with rows of their own end by themselves
  for (int turn = 0; row < a.rows; row += step, turn ^= 1) {
    float xv[K][VN], rv[K][VN], sg[K][VN], zv[K][VN], ov[K][VN], ss = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        xv[k][e] = xr[k].get(e);
        rv[k][e] = rr[k].get(e);
        sg[k][e] = gr[k].get(e);
        zv[k][e] = zr[k].get(e);
        ov[k][e] = orr[k].get(e);
        ss += xv[k][e] * xv[k][e];
      }
    fetch(row + step);
    float rho = 1.f;
    if (a.post) rho = rsqrtf(row_sum<TPR>(ss, red[turn][0]) * a.inv_d + a.eps);
    float rss = 0.f, dot = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        sg[k][e] = a.gate ? sigmoid(sg[k][e]) : 1.f;
        rv[k][e] += xv[k][e] * rho * cp[k][e] * sg[k][e];
        rss += rv[k][e] * rv[k][e];
        dot += zv[k][e] * wv[k][e] * rv[k][e];
      }
    if (a.dz) {
      row_sum2<TPR>(rss, dot, red[turn][1]);
      const float rho2 = rsqrtf(rss * a.inv_d + a.eps), m = dot * a.inv_d * rho2 * rho2;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          ov[k][e] += rho2 * (zv[k][e] * wv[k][e] - rv[k][e] * m);
          dw[k][e] += zv[k][e] * rv[k][e] * rho2;
        }
    }
    const int64_t base = row * a.d;
    dot = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = first_column<TPR, VN, ES>(k, li), left = a.d - c;
      if (a.dr && left > 0) store_row<S, VN, ES>(static_cast<S*>(a.dr) + base + c, left, ov[k]);
      float dg[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const float xn = xv[k][e] * rho;
        db[k][e] += ov[k][e] * sg[k][e] * xn;
        ov[k][e] *= cp[k][e] * sg[k][e];  // v
        dg[e] = ov[k][e] * xn * (1.f - sg[k][e]);
        dot += ov[k][e] * xv[k][e];
      }
      if (a.dgate && left > 0) store_row<G, VN, ES>(static_cast<G*>(a.dgate) + base + c, left, dg);
    }
    float m = 0.f;
    if (a.post) m = row_sum<TPR>(dot, red[turn][2]) * a.inv_d * rho * rho;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = first_column<TPR, VN, ES>(k, li), left = a.d - c;
#pragma unroll
      for (int e = 0; e < VN; ++e) ov[k][e] = a.post ? rho * (ov[k][e] - xv[k][e] * m) : ov[k][e];  // (an infinite x times m = 0 is no 0)
      if (left > 0) store_row<T, VN, ES>(static_cast<T*>(a.dx) + base + c, left, ov[k]);
    }
  }
  if (!a.dw) return;
  // one partial row of both sums per workgroup: [d_weight | S], dpad columns each
  float* part = a.dw + (int64_t)blockIdx.x * 2 * a.dpad;
  if constexpr (RPB > 1) {
    __shared__ float sums[RPB - 1][2][C];
    if (sub > 0) {
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const int c = (k * TPR + li) * VN + e;
          sums[sub - 1][0][c] = dw[k][e];
          sums[sub - 1][1][c] = db[k][e];
        }
    }
    __syncthreads();
    if (sub > 0) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const int c = (k * TPR + li) * VN + e;
#pragma unroll
        for (int s = 0; s < RPB - 1; ++s) dw[k][e] += sums[s][0][c], db[k][e] += sums[s][1][c];
      }
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < VN; e += VEC ? 4 : 1) {
      const int c = first_column<TPR, VN, ES>(k, li) + e * ES;
      if (c >= a.dpad) continue;
      if constexpr (!VEC) {
        part[c] = dw[k][e];
        part[a.dpad + c] = db[k][e];
      } else {
        store4(part + c, floatx4{dw[k][e], dw[k][e + 1], dw[k][e + 2], dw[k][e + 3]});
        store4(part + a.dpad + c, floatx4{db[k][e], db[k][e + 1], db[k][e + 2], db[k][e + 3]});
      }
    }
}

// Adds the partial rows: 16 columns a workgroup, 64 sets of rows, eight loads in flight a thread; d_post = scale S, d_scale = post S.
__global__ __launch_bounds__(256) void rmsnorm_residual_sums_kernel(const float* part, int n, int d, int dpad, const float* post, const float* scale_v, float scale,
                                                                    float* d_weight, float* d_post, float* d_scale) {
  __shared__ floatx4 red[64][4];
  const int cg = threadIdx.x & 3, rs = threadIdx.x >> 2;
  const int c = (blockIdx.x * 4 + cg) * 4;  // of 2 dpad columns
  floatx4 acc[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) acc[u] = floatx4{0.f, 0.f, 0.f, 0.f};
  if (c < 2 * dpad)
    for (int r = rs; r < n; r += 64 * 8)
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r + 64 * u < n) acc[u] += load4(part + (int64_t)(r + 64 * u) * 2 * dpad + c);
  red[rs][cg] = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
  for (int s = 32; s >= 1; s >>= 1) {
    __syncthreads();
    if (rs < s) red[rs][cg] += red[rs + s][cg];
  }
  if (rs != 0 || c >= 2 * dpad) return;
  const floatx4 t = red[0][cg];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bool first = c < dpad;
    const int col = (first ? c : c - dpad) + e;
    if (col >= d) continue;
    if (first) {
      if (d_weight) d_weight[col] = t[e];
    } else {
      if (d_post) d_post[col] = t[e] * (scale_v ? scale_v[col] : scale);
      if (d_scale) d_scale[col] = t[e] * (post ? post[col] : 1.f);
    }
  }
}

// Threads and vectors per row: one wave up to two vectors a lane, then workgroups of 256 and 512
struct Plan { int tpr, k; };
Plan plan(int d, int dtype) {
  const int vn = dtype == LNX_BF16 ? 8 : 4, v = (d + vn - 1) / vn;
  if (v <= 64) return {64, 1};
  if (v <= 128) return {64, 2};
  if (v <= 256) return {256, 1};
  if (v <= 512) return {256, 2};
  if (v <= 1024) return {512, 2};
  return {512, 4};  // fp32 only: eight vectors of bf16 a thread would not fit the backward pass's registers
}
constexpr int MAX_D = 8192;

// Workgroups of the backward pass: three a CU, each with one partial row of the parameters' gradients
int bwd_blocks(int64_t rows, const Plan& p) {
  const int64_t rpb = block_of(p.tpr) / p.tpr, all = (rows + rpb - 1) / rpb;
  return (int)(all < 768 ? all : 768);
}

template <typename T, typename S, typename G, int TPR, int K> void launch(const Args& a, bool vec, bool bwd, int blocks, hipStream_t st) {
  const int wide = blocks < 1 << 22 ? blocks : 1 << 22;  // a launch takes 2^32 threads in one direction
  const dim3 g((unsigned)wide, (unsigned)((blocks + wide - 1) / wide)), b(block_of(TPR));
  if (bwd) {
    if (vec) rmsnorm_residual_bwd_kernel<T, S, G, TPR, K, true><<<g, b, 0, st>>>(a);
    else rmsnorm_residual_bwd_kernel<T, S, G, TPR, K, false><<<g, b, 0, st>>>(a);
  } else {
    if (vec) rmsnorm_residual_fwd_kernel<T, S, G, TPR, K, true><<<g, b, 0, st>>>(a);
    else rmsnorm_residual_fwd_kernel<T, S, G, TPR, K, false><<<g, b, 0, st>>>(a);
  }
}

template <typename T, typename S, typename G> void pick(const Args& a, const Plan& p, bool vec, bool bwd, int blocks, hipStream_t st) {
  if (p.tpr == 64 && p.k == 1) launch<T, S, G, 64, 1>(a, vec, bwd, blocks, st);
  else if (p.tpr == 64) launch<T, S, G, 64, 2>(a, vec, bwd, blocks, st);
  else if (p.tpr == 256 && p.k == 1) launch<T, S, G, 256, 1>(a, vec, bwd, blocks, st);
  else if (p.tpr == 256) launch<T, S, G, 256, 2>(a, vec, bwd, blocks, st);
  else if (p.k == 2) launch<T, S, G, 512, 2>(a, vec, bwd, blocks, st);
  else if constexpr (sizeof(T) == 4) launch<T, S, G, 512, 4>(a, vec, bwd, blocks, st);
}

int run(const char* what, const lnx_rmsnorm_residual_args* q, bool bwd, hipStream_t st) {
  if (!q) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (q->rows < 0 || q->rows > 0x7fffffff || q->d <= 0 || q->d > MAX_D)
    return lnx_set_error(LNX_ERR_SHAPE, "%s: rows=%lld d=%d (at most %d columns)", what, (long long)q->rows, q->d, MAX_D);
  if ((q->dtype != LNX_F32 && q->dtype != LNX_BF16) || (q->r_dtype != LNX_F32 && q->r_dtype != q->dtype))
    return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d, r_dtype %d (x float32 or bfloat16, the residual float32 or x's type)", what, q->dtype, q->r_dtype);
  if (q->rows > 0 && !q->x) return lnx_set_error(LNX_ERR_NULL, "%s: x is required", what);
  const bool params = bwd && (q->d_weight || q->d_post_weight || q->d_scale);
  if (!bwd && q->rows > 0 && (!q->out || (q->z && !q->weight))) return lnx_set_error(LNX_ERR_NULL, "%s: out (and weight for z) is required", what);
  if (bwd && q->rows > 0 && (!q->d_x || (q->gate && !q->d_gate) || (q->d_z && !q->weight)))
    return lnx_set_error(LNX_ERR_NULL, "%s: d_x (d_gate with a gate, weight with d_z) is required", what);
  if (params && (!q->workspace || reinterpret_cast<uintptr_t>(q->workspace) % 16 || q->workspace_bytes < lnx_rmsnorm_residual_bwd_workspace_bytes(q->rows, q->d, q->dtype)))
    return lnx_set_error(LNX_ERR_WORKSPACE, "%s: the parameters' gradients need a 16-byte aligned workspace of %llu bytes", what,
                         (unsigned long long)lnx_rmsnorm_residual_bwd_workspace_bytes(q->rows, q->d, q->dtype));
  if (q->rows == 0 && !params) return LNX_OK;
  Args a{};
  a.x = q->x, a.r = q->residual, a.gate = q->gate, a.w = q->weight, a.post = q->post_weight, a.scale_v = q->scale_vector;
  a.scale = q->scale, a.eps = q->eps, a.inv_d = 1.f / (float)q->d, a.rows = q->rows, a.d = q->d, a.dpad = (q->d + 3) / 4 * 4;
  a.z = q->z, a.out = q->out;
  a.dz = q->d_z, a.dout = q->d_out, a.dx = q->d_x, a.dr = q->residual ? q->d_residual : nullptr, a.dgate = q->d_gate;
  const int vn = q->dtype == LNX_BF16 ? 8 : 4;
  bool vec = q->d % vn == 0;
  for (const void* p : {a.x, a.r, a.gate, (const void*)a.w, (const void*)a.post, (const void*)a.scale_v, (const void*)a.z, (const void*)a.out, a.dz, a.dout,
                        (const void*)a.dx, (const void*)a.dr, (const void*)a.dgate})
    vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  const Plan p = plan(q->d, q->dtype);
  int blocks = 0;
  if (q->rows > 0) {
    const int64_t rpb = block_of(p.tpr) / p.tpr;
    blocks = bwd ? bwd_blocks(q->rows, p) : (int)((q->rows + rpb - 1) / rpb);
    if (params) a.dw = static_cast<float*>(q->workspace);
    lnx_profile_mark(what, st);
    const bool wide = q->gate && q->gate_f32;  // a gate of its own type beside bf16
    if (q->dtype == LNX_F32) pick<float, float, float>(a, p, vec, bwd, blocks, st);
    else if (q->r_dtype == LNX_F32) wide ? pick<bf16_t, float, float>(a, p, vec, bwd, blocks, st) : pick<bf16_t, float, bf16_t>(a, p, vec, bwd, blocks, st);
    else wide ? pick<bf16_t, bf16_t, float>(a, p, vec, bwd, blocks, st) : pick<bf16_t, bf16_t, bf16_t>(a, p, vec, bwd, blocks, st);
  }
  if (params) {
    lnx_profile_mark("rmsnorm_residual_sums", st);
    rmsnorm_residual_sums_kernel<<<dim3((unsigned)((2 * a.dpad + 15) / 16)), 256, 0, st>>>(static_cast<const float*>(q->workspace), blocks, q->d, a.dpad, a.post, a.scale_v,
                                                                                          a.scale, q->d_weight, q->d_post_weight, q->d_scale);
  }
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" uint64_t lnx_rmsnorm_residual_bwd_workspace_bytes(int64_t rows, int32_t d, int32_t dtype) {
  if (rows < 0 || d <= 0 || d > MAX_D) return 0;
  const Plan p = plan(d, dtype);
  const int n = bwd_blocks(rows, p);
  return (uint64_t)(n > 0 ? n : 1) * 2 * ((d + 3) / 4 * 4) * sizeof(float);
}

extern "C" int lnx_rmsnorm_residual_fwd(const lnx_rmsnorm_residual_args* a, void* hip_stream) {
  return run("rmsnorm_residual_fwd", a, false, static_cast<hipStream_t>(hip_stream));
}
extern "C" int lnx_rmsnorm_residual_bwd(const lnx_rmsnorm_residual_args* a, void* hip_stream) {
  return run("rmsnorm_residual_bwd", a, true, static_cast<hipStream_t>(hip_stream));
}
