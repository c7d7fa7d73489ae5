// Layer norm over the last dimension, forward and backward, with weights [d] or one set for each of n heads ([n, d] under rows [.., n, d]):
//   mean = sum x / d    rho = (sum (x - mean)^2 / d + eps)^(-1/2)    h = (x - mean) rho    y = h w + b
//   u = dy w    dx = rho (u - sum u / d - h (sum u h) / d)    dw = sum dy h    db = sum dy
// Bound by bytes: a row (or several) is read once with 16-byte loads and stays in registers between its reductions; the variance is a second
// sum over the registers.  A mean far from zero is off by units of itself, which the differences carry: they are summed beside their squares, and
// what their own mean misses is taken off (rows of 768 around 10^4 with a deviation of 2: y off by 4.8e-4 -> 4.3e-7, dx 5e-5 -> 4e-7; a per cent of the backward
// pass's time).  The backward pass forms mean and rho again from x, which it needs anyway: nothing is kept.  Its sums over the rows stay in registers over all rows of a workgroup, which are rows of one head, and
// leave as one partial row each; a second launch adds them (no atomics, the same from run to run).
// 32768 rows of 2048 in bf16: forward 57 - 60 us, 4.5 - 4.7 TB/s, backward 82 - 93 (403 MB) and 7 for the sums; 32768 x 16 heads of 128: 46 - 49, 80 - 82,
// 5.  A group of TPR lanes takes four rows at a time where there are workgroups enough (heads of 128: forward 55 us with one row).
#include "lnx_common.h"
#include "mma_tiles.h"
#include "reduce_rows.h"
#include "row_vectors.h"

namespace {

struct Args {
  const void *x, *dy;
  const float *w, *b;
  void *y, *dx;
  float* part;    // partial rows [block][dw | db], dpad columns each
  int64_t outer;  // rows of a head
  int d, dpad, n;
  float eps, inv_d;
};

constexpr int block_of(int tpr) { return tpr < 256 ? 256 : tpr; }

template <int K, int VN> struct Columns {
  float v[K][VN];
  __device__ __forceinline__ void fill(float f) {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) v[k][e] = f;
  }
};
template <int TPR, int K, int VN, int ES> __device__ __forceinline__ void load_columns(Columns<K, VN>& c, const float* p, int d, int li, float absent) {
  c.fill(p ? 0.f : absent);
  if (!p) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int at = first_column<TPR, VN, ES>(k, li);
    if (at < d) load_row<float, VN, ES>(p + at, d - at, c.v[k]);
  }
}

// x less the row's mean, opaque: -ffast-math would form the sum of the differences from the sums that they are to mend
__device__ __forceinline__ float centred(float x, float mean) {
  x -= mean;
  asm("" : "+v"(x));
  return x;
}
// 1 / sqrt(var + eps) from the mean of the squared differences and their own mean
__device__ __forceinline__ float inv_std(float square, float miss, float eps) { return rsqrtf(fmaxf(square - miss * miss, 0.f) + eps); }

// Whether element e of a thread's k-th vector is a column of the row
template <int TPR, int VN, int ES> __device__ __forceinline__ bool inside(int k, int e, int li, int d) { return first_column<TPR, VN, ES>(k, li) + e * ES < d; }

// Workgroup = (block of rows, head), heads next to each other; every group of TPR threads takes U rows, all on their way before the first is used.
template <typename T, int TPR, int K, bool VEC, int U> __global__ __launch_bounds__(block_of(TPR)) void layer_norm_fwd_kernel(Args a) {
  constexpr int VN = Vec16<T>::N, RPB = block_of(TPR) / TPR, ES = VEC ? 1 : TPR;
  static_assert(U == 1 || TPR <= 64, "rows of several waves share their slots for sums");
  __shared__ float red[2][32];
  const int li = threadIdx.x % TPR;
  const int64_t blk = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int head = (int)(blk % a.n);
  const int64_t row0 = blk / a.n * (RPB * U) + threadIdx.x / TPR;
  if (row0 >= a.outer) return;  // whole rows; those of up to a wave have no barrier, of longer ones a workgroup has one
  RawRow<T, VN, ES> xr[U][K];
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int64_t row = row0 + u * RPB;
      const int c = first_column<TPR, VN, ES>(k, li);
      xr[u][k].load(static_cast<const T*>(a.x) + (row * a.n + head) * a.d + c, row < a.outer ? a.d - c : 0);
    }
  Columns<K, VN> w, b;
  load_columns<TPR, K, VN, ES>(w, a.w ? a.w + (int64_t)head * a.d : nullptr, a.d, li, 1.f);
  load_columns<TPR, K, VN, ES>(b, a.b ? a.b + (int64_t)head * a.d : nullptr, a.d, li, 0.f);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t row = row0 + u * RPB;
    float xv[K][VN], s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) s += xv[k][e] = xr[u][k].get(e);
    const float mean = row_sum<TPR>(s, red[0]) * a.inv_d;
    float sums[2] = {0.f, 0.f};  // of the differences' squares, of themselves
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        xv[k][e] = inside<TPR, VN, ES>(k, e, li, a.d) ? centred(xv[k][e], mean) : 0.f;
        sums[0] += xv[k][e] * xv[k][e];
        sums[1] += xv[k][e];
      }
    row_sums<TPR>(sums, red[1]);
    const float miss = sums[1] * a.inv_d, rho = inv_std(sums[0] * a.inv_d, miss, a.eps), off = miss * rho;
    if (row >= a.outer) return;
    T* y = static_cast<T*>(a.y) + (row * a.n + head) * a.d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = first_column<TPR, VN, ES>(k, li);
#pragma unroll
      for (int e = 0; e < VN; ++e) xv[k][e] = (xv[k][e] * rho - off) * w.v[k][e] + b.v[k][e];
      if (c < a.d) store_row<T, VN, ES>(y + c, a.d - c, xv[k]);
    }
  }
}

// Rows of one head, gridDim.x / n workgroups apart; the next row is on its way while one is worked on.
template <typename T, int TPR, int K, bool VEC> __global__ __launch_bounds__(block_of(TPR)) void layer_norm_bwd_kernel(Args a) {
  constexpr int VN = Vec16<T>::N, RPB = block_of(TPR) / TPR, C = TPR * K * VN, ES = VEC ? 1 : TPR;
  __shared__ float red[2][2][48];
  const int li = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int head = (int)(blockIdx.x % a.n);
  Columns<K, VN> w, dw, db;
  load_columns<TPR, K, VN, ES>(w, a.w ? a.w + (int64_t)head * a.d : nullptr, a.d, li, 1.f);
  dw.fill(0.f);
  db.fill(0.f);
  RawRow<T, VN, ES> xr[K], gr[K];
  const auto fetch = [&](int64_t row) {
    const int64_t base = (row * a.n + head) * a.d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = first_column<TPR, VN, ES>(k, li), left = row < a.outer ? a.d - c : 0;
      xr[k].load(static_cast<const T*>(a.x) + base + c, left);
      gr[k].load(static_cast<const T*>(a.dy) + base + c, left);
    }
  };
  const int64_t step = (int64_t)(gridDim.x / a.n) * RPB;
  int64_t row = (int64_t)(blockIdx.x / a.n) * RPB + sub;
  fetch(row);
  // every thread of a workgroup of one row takes the same number of turns (barriers); parts of a wave go on by themselves
  for (int turn = 0; row < a.outer; row += step, turn ^= 1) {
    float xv[K][VN], uv[K][VN], first[2] = {0.f, 0.f}, sums[3] = {0.f, 0.f, 0.f};  // of x, u; of the differences' squares, u times them, themselves
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        first[0] += xv[k][e] = xr[k].get(e);
        uv[k][e] = gr[k].get(e);
        db.v[k][e] += uv[k][e];
        first[1] += uv[k][e] * w.v[k][e];
      }
    fetch(row + step);
    row_sums<TPR>(first, red[turn][0]);
    const float mean = first[0] * a.inv_d, mu = first[1] * a.inv_d;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        xv[k][e] = inside<TPR, VN, ES>(k, e, li, a.d) ? centred(xv[k][e], mean) : 0.f;
        sums[0] += xv[k][e] * xv[k][e];
        sums[1] += uv[k][e] * w.v[k][e] * xv[k][e];
        sums[2] += xv[k][e];
      }
    row_sums<TPR>(sums, red[turn][1]);
    const float miss = sums[2] * a.inv_d, rho = inv_std(sums[0] * a.inv_d, miss, a.eps), off = miss * rho, m = (sums[1] * a.inv_d - miss * mu) * rho * rho, shift = mu - miss * m;
    T* dx = static_cast<T*>(a.dx) + (row * a.n + head) * a.d;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = first_column<TPR, VN, ES>(k, li);
      float o[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        dw.v[k][e] += uv[k][e] * (xv[k][e] * rho - off);
        o[e] = rho * (uv[k][e] * w.v[k][e] - shift - xv[k][e] * m);
      }
      if (c < a.d) store_row<T, VN, ES>(dx + c, a.d - c, o);
    }
  }
  if (!a.part) return;
  float* part = a.part + (int64_t)blockIdx.x * 2 * a.dpad;
  if constexpr (RPB > 1) {  // the workgroup's rows: by halves
    __shared__ float sums[RPB / 2][2][C];
    for (int half = RPB / 2; half >= 1; half >>= 1) {
      if (sub >= half && sub < 2 * half)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            const int c = (k * VN + e) * TPR + li;
            sums[sub - half][0][c] = dw.v[k][e];
            sums[sub - half][1][c] = db.v[k][e];
          }
      __syncthreads();
      if (sub < half)
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            const int c = (k * VN + e) * TPR + li;
            dw.v[k][e] += sums[sub][0][c];
            db.v[k][e] += sums[sub][1][c];
          }
      __syncthreads();
    }
    if (sub > 0) return;
  }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int e = 0; e < VN; e += VEC ? 4 : 1) {
      const int c = first_column<TPR, VN, ES>(k, li) + e * ES;
      if (c >= a.dpad) continue;
      if constexpr (!VEC) {
        part[c] = dw.v[k][e];
        part[a.dpad + c] = db.v[k][e];
      } else {
        store4(part + c, floatx4{dw.v[k][e], dw.v[k][e + 1], dw.v[k][e + 2], dw.v[k][e + 3]});
        store4(part + a.dpad + c, floatx4{db.v[k][e], db.v[k][e + 1], db.v[k][e + 2], db.v[k][e + 3]});
      }
    }
}

// Adds the `per` partial rows of every head: 16 columns a workgroup, 64 sets of rows, eight loads in flight a thread.
__global__ __launch_bounds__(256) void layer_norm_sums_kernel(const float* part, int per, int n, int d, int dpad, float* d_weight, float* d_bias) {
  __shared__ floatx4 red[64][4];
  const int cg = threadIdx.x & 3, rs = threadIdx.x >> 2, width = 2 * dpad, tiles = (width + 15) / 16;
  const int head = blockIdx.x / tiles, c = ((blockIdx.x % tiles) * 4 + cg) * 4;  // of the head's 2 dpad columns
  floatx4 acc[8];
#pragma unroll
  for (int u = 0; u < 8; ++u) acc[u] = floatx4{0.f, 0.f, 0.f, 0.f};
  if (c < width)
    for (int r = rs; r < per; r += 64 * 8)
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (r + 64 * u < per) acc[u] += load4(part + ((int64_t)(r + 64 * u) * n + head) * width + c);
  red[rs][cg] = ((acc[0] + acc[1]) + (acc[2] + acc[3])) + ((acc[4] + acc[5]) + (acc[6] + acc[7]));
  for (int s = 32; s >= 1; s >>= 1) {
    __syncthreads();
    if (rs < s) red[rs][cg] += red[rs + s][cg];
  }
  if (rs != 0 || c >= width) return;
  const floatx4 t = red[0][cg];
  const bool first = c < dpad;
  float* out = first ? d_weight : d_bias;
  if (!out) return;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int col = (first ? c : c - dpad) + e;
    if (col < d) out[(int64_t)head * d + col] = t[e];
  }
}

// Threads and vectors per row: as few lanes as hold it, a wave up to two vectors a lane, then workgroups of 256 and 512
struct Plan { int tpr, k; };
Plan plan(int d, int dtype) {
  const int vn = dtype == LNX_BF16 ? 8 : 4, v = (d + vn - 1) / vn;
  if (v <= 8) return {8, 1};
  if (v <= 16) return {16, 1};
  if (v <= 32) return {32, 1};
  if (v <= 64) return {64, 1};
  if (v <= 128) return {64, 2};
  if (v <= 256) return {256, 1};
  if (v <= 512) return {256, 2};
  if (v <= 1024) return {512, 2};
  return {512, 4};  // fp32 only: eight vectors of bf16 a thread would not fit the backward pass's registers
}
constexpr int MAX_D = 8192, MAX_HEADS = 1 << 16, MAX_WEIGHTS = 1 << 26;  // the last: the sums' launch takes 16 threads a column

// Workgroups of the backward pass per head: three a CU in all, each with one partial row of the parameters' gradients
int64_t bwd_per_head(int64_t outer, int64_t n, const Plan& p) {
  const int64_t rpb = block_of(p.tpr) / p.tpr, all = (outer + rpb - 1) / rpb, most = (768 + n - 1) / n;
  return all < most ? all : most;
}

template <typename T, int TPR, int K> void launch(const Args& a, bool vec, bool bwd, int64_t bwd_blocks, hipStream_t st) {
  constexpr int RPB = block_of(TPR) / TPR, MANY = TPR <= 64 ? 4 : 1;
  const dim3 b(block_of(TPR));
  if (bwd) {
    const dim3 g((unsigned)bwd_blocks);
    if (vec) layer_norm_bwd_kernel<T, TPR, K, true><<<g, b, 0, st>>>(a);
    else layer_norm_bwd_kernel<T, TPR, K, false><<<g, b, 0, st>>>(a);
    return;
  }
  const int64_t one = (a.outer + RPB - 1) / RPB * a.n;
  const bool many = MANY > 1 && one >= 8192;
  const int64_t blocks = many ? (a.outer + RPB * MANY - 1) / (RPB * MANY) * a.n : one;
  const int64_t wide = blocks < 1 << 22 ? blocks : 1 << 22;  // a launch takes 2^32 threads in one direction
  const dim3 g((unsigned)wide, (unsigned)((blocks + wide - 1) / wide));
  if (many) {
    if (vec) layer_norm_fwd_kernel<T, TPR, K, true, MANY><<<g, b, 0, st>>>(a);
    else layer_norm_fwd_kernel<T, TPR, K, false, MANY><<<g, b, 0, st>>>(a);
  } else {
    if (vec) layer_norm_fwd_kernel<T, TPR, K, true, 1><<<g, b, 0, st>>>(a);
    else layer_norm_fwd_kernel<T, TPR, K, false, 1><<<g, b, 0, st>>>(a);
  }
}

template <typename T> void pick(const Args& a, const Plan& p, bool vec, bool bwd, int64_t bwd_blocks, hipStream_t st) {
  if (p.tpr == 8) launch<T, 8, 1>(a, vec, bwd, bwd_blocks, st);
  else if (p.tpr == 16) launch<T, 16, 1>(a, vec, bwd, bwd_blocks, st);
  else if (p.tpr == 32) launch<T, 32, 1>(a, vec, bwd, bwd_blocks, st);
  else if (p.tpr == 64 && p.k == 1) launch<T, 64, 1>(a, vec, bwd, bwd_blocks, st);
  else if (p.tpr == 64) launch<T, 64, 2>(a, vec, bwd, bwd_blocks, st);
  else if (p.tpr == 256 && p.k == 1) launch<T, 256, 1>(a, vec, bwd, bwd_blocks, st);
  else if (p.tpr == 256) launch<T, 256, 2>(a, vec, bwd, bwd_blocks, st);
  else if (p.k == 2) launch<T, 512, 2>(a, vec, bwd, bwd_blocks, st);
  else if constexpr (sizeof(T) == 4) launch<T, 512, 4>(a, vec, bwd, bwd_blocks, st);
}

int run(const char* what, const lnx_layer_norm_args* q, bool bwd, hipStream_t st) {
  if (!q) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (q->rows < 0 || q->rows > 0x7fffffff || q->d <= 0 || q->d > MAX_D || q->heads <= 0 || q->heads > MAX_HEADS || (int64_t)q->heads * q->d > MAX_WEIGHTS || q->rows % q->heads)
    return lnx_set_error(LNX_ERR_SHAPE, "%s: rows=%lld heads=%d d=%d (at most %d columns, %d heads, %d weights; rows a multiple of heads)", what, (long long)q->rows, q->heads,
                         q->d, MAX_D, MAX_HEADS, MAX_WEIGHTS);
  if (q->dtype != LNX_F32 && q->dtype != LNX_BF16) return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d", what, q->dtype);
  if (q->rows > 0 && (!q->x || (bwd ? !q->d_y || !q->d_x : !q->y))) return lnx_set_error(LNX_ERR_NULL, "%s: %s required", what, bwd ? "x, d_y and d_x are" : "x and y are");
  const bool params = bwd && (q->d_weight || q->d_bias);
  const uint64_t need = params ? lnx_layer_norm_bwd_workspace_bytes(q->rows, q->heads, q->d, q->dtype) : 0;
  if (params && (!q->workspace || reinterpret_cast<uintptr_t>(q->workspace) % 16 || q->workspace_bytes < need))
    return lnx_set_error(LNX_ERR_WORKSPACE, "%s: the parameters' gradients need a 16-byte aligned workspace of %llu bytes", what, (unsigned long long)need);
  if (q->rows == 0 && !params) return LNX_OK;
  Args a{};
  a.x = q->x, a.dy = q->d_y, a.w = q->weight, a.b = q->bias, a.y = q->y, a.dx = q->d_x;
  a.outer = q->rows / q->heads, a.d = q->d, a.dpad = (q->d + 3) / 4 * 4, a.n = q->heads, a.eps = q->eps, a.inv_d = 1.f / (float)q->d;
  bool vec = q->d % (q->dtype == LNX_BF16 ? 8 : 4) == 0;
  for (const void* p : {a.x, a.dy, (const void*)a.w, (const void*)a.b, (const void*)a.y, (const void*)a.dx}) vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
  const Plan p = plan(q->d, q->dtype);
  const int64_t per = bwd_per_head(a.outer, a.n, p);
  if (q->rows > 0) {
    if (params) a.part = static_cast<float*>(q->workspace);
    lnx_profile_mark(what, st);
    if (q->dtype == LNX_F32) pick<float>(a, p, vec, bwd, per * a.n, st);
    else pick<bf16_t>(a, p, vec, bwd, per * a.n, st);
  }
  if (params) {
    lnx_profile_mark("layer_norm_sums", st);
    layer_norm_sums_kernel<<<dim3((unsigned)((2 * a.dpad + 15) / 16 * a.n)), 256, 0, st>>>(static_cast<const float*>(q->workspace), (int)per, a.n, a.d, a.dpad, q->d_weight, q->d_bias);
  }
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" uint64_t lnx_layer_norm_bwd_workspace_bytes(int64_t rows, int32_t heads, int32_t d, int32_t dtype) {
  if (rows < 0 || heads <= 0 || heads > MAX_HEADS || d <= 0 || d > MAX_D) return 0;
  const int64_t per = bwd_per_head(rows / heads, heads, plan(d, dtype));
  return (uint64_t)(per > 0 ? per : 1) * heads * 2 * ((d + 3) / 4 * 4) * sizeof(float);
}
extern "C" int lnx_layer_norm_fwd(const lnx_layer_norm_args* a, void* hip_stream) { return run("layer_norm_fwd", a, false, static_cast<hipStream_t>(hip_stream)); }
extern "C" int lnx_layer_norm_bwd(const lnx_layer_norm_args* a, void* hip_stream) { return run("layer_norm_bwd", a, true, static_cast<hipStream_t>(hip_stream)); }
