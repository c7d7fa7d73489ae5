// Causal softmax attention over whole prompts, grouped heads, dense or packed, forward and backward on the matrix cores:
//   s_ij = scale q_i . k_j   p_ij = exp(s_ij - lse_i)  (j <= i)   o_i = sum_j p_ij v_j
//   delta_i = o_i . do_i   ds_ij = p_ij (do_i . v_j - delta_i)   dq_i = scale sum_j ds_ij k_j   dk_j = scale sum_i ds_ij q_i   dv_j = sum_i p_ij do_i
// One pass over the keys with running maximum and sum; no score ever leaves the registers.  Every product is laid out so that its
// result fragment is the next product's operand as it is: a wave owns 32 columns -- queries in the forward and the dq kernel, keys in
// the dk / dv kernel -- whose vectors stay in registers as B operands, and the rows that it walks over lie in LDS, read by rows for
// the products over the head dimension and through transposing reads for the products over the rows.  A score fragment holds one
// column per lane and half, so maxima and sums are within the lane and one exchange of the wave's halves.
// Tiles of 64 rows (32 in the bf16 forward kernel at d > 64) come in through loads that go straight to LDS, the next tile behind the one being
// multiplied, one barrier a tile.
// bf16 takes v_mfma_f32_32x32x16_bf16 (probabilities and score gradients are rounded to bf16 as operands: at most 2^-8 of each term, what
// the outputs are rounded to; all in all 0.0024 of the norm for a training step and 0.0021 for a prompt, where the rounding of the results alone
// is 0.0017 and 0.0016; in two parts, with up to half of the products more, it is that alone: see SHORT), fp32 takes v_mfma_f32_32x32x2_f32
// throughout.  Sums, maxima and accumulators are fp32.
// Bound by the matrix cores and the exponentials beside them: at B2 H16/4 T4096 d128 bf16 the forward kernel takes 147-164 us (840-930
// TFLOP/s of the causal half), dq 194-217, dk / dv 311-343 and the two sums of its parts 7 each, together 600-650 TFLOP/s of the 10 d operations a
// pair that the gradient needs (scores and do . v are formed in both kernels, 14 d in all), where a large library product reaches 1200.  Matrix cores
// are busy 44, 45 and 36 % of the time, vector instructions 50, 33 and 26 %.
// No atomics: dk and dv are summed over the group's query heads by the workgroup that owns the keys, dq by a kernel of its own.
#include "lnx_common.h"
#include "mma_tiles.h"
#include "packed_slots.h"

namespace {

constexpr int ROWS = 64;  // rows of a tile
constexpr int64_t MAX_GRID = 0xffffffff / 256;  // workgroups of a launch
constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ unsigned fresh(unsigned x) { return (unsigned)::fresh((int)x); }

struct Args {
  const void *q, *k, *v, *dout;
  void *o, *o_low, *dq, *dk, *dv;  // o_low [B, H, T, d]: what o's rounding left
  float *lse, *delta;  // [B, H, T]; lse in units of log 2
  const int32_t* cu;
  int64_t qs[3], ks[3], vs[3], os[3], gs[3], dqs[3], dks[3], dvs[3];  // strides of batch, head, token in elements
  float *part, *part_stat;  // shares of workgroups that split a block's rows between them: [parts][rows of the result][d], [parts][rows][2]
  int B, H, Hkv, G, T, d, nseq, nblk, parts;
  float scale;
};

// Eight contraction slots of an operand
template <typename T> struct Frag8;
template <> struct Frag8<bf16_t> {
  bf16x8 v;
  __device__ __forceinline__ void zero() { v = vec_zero<bf16_t>(); }
};
template <> struct Frag8<float> {
  float v[8];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
  }
};
__device__ __forceinline__ void mma(floatx16& c, const Frag8<bf16_t>& a, const Frag8<bf16_t>& b) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.v, b.v, c, 0, 0, 0); }
__device__ __forceinline__ void mma(floatx16& c, const Frag8<float>& a, const Frag8<float>& b) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[e], b.v[e], c, 0, 0, 0);
}
// Elements 8 h .. 8 h + 7 of a result fragment as an operand in chain order (rows 16 h + 4 kg + 0 .. 3 and + 8 .. 11)
__device__ __forceinline__ void from_acc(Frag8<bf16_t>& f, const floatx16& c, int h) { f.v = Mma<bf16_t>::from_acc(c, h); }
__device__ __forceinline__ void from_acc(Frag8<float>& f, const floatx16& c, int h) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f.v[e] = c[8 * h + e];
}
// Eight consecutive elements from memory; `ok`: they exist
template <typename T> __device__ __forceinline__ void from_global(Frag8<T>& f, const T* p, bool ok);
template <> __device__ __forceinline__ void from_global<bf16_t>(Frag8<bf16_t>& f, const bf16_t* p, bool ok) {
  f.zero();
  if (ok) f.v = *reinterpret_cast<const bf16x8*>(p);
}
template <> __device__ __forceinline__ void from_global<float>(Frag8<float>& f, const float* p, bool ok) {
  f.zero();
  if (ok) {
    const floatx4 a = load4(p), b = load4(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) f.v[e] = a[e], f.v[e + 4] = b[e];
  }
}

// A [R][D] tile in LDS, 16-byte granules of a row permuted by an exclusive or with the row, so that row reads and reads along the rows
// spread over the banks.  A lane reads at an address of its own exclusive-or a constant per column block, plus a constant per
// block of rows that fits the instruction's offset: rows() and cols() give the lane's addresses, by_row and by_col the operands.
typedef __attribute__((address_space(3))) char lds_char;
template <typename V> __device__ __forceinline__ V lds_load(unsigned addr) { return *(__attribute__((address_space(3))) const V*)(lds_char*)(uintptr_t)addr; }

template <typename T, int D, int R = ROWS> struct Tile;
template <int D, int R> struct Tile<bf16_t, D, R> {
  typedef SwzTile<R, D> S;
  static constexpr int BYTES = R * D * 2, ROWB = D * 2;
  static __device__ __forceinline__ void src(int j, int lane, int& r, int& c) { S::src(j, lane, r, c); }
  // rows r = lane & 31 of 32, columns 16 s + 8 kg + 0 .. 7: granule (2 s + kg) ^ x(r)
  static __device__ __forceinline__ unsigned rows(int lane) { return 2 * S::at(lane & 31, 8 * (lane >> 5)); }
  static __device__ __forceinline__ Frag8<bf16_t> by_row(unsigned rows, int off, int s) { return {lds_load<bf16x8>((rows ^ (32 * s)) + off)}; }
  // rows 4 kg + 0 .. 3 and 8 + 4 kg + 0 .. 3 of 16, column 32 m + (lane & 31): two transposing reads of four rows each
  static __device__ __forceinline__ unsigned cols(int lane) {
    const int s = lane & 15, grp = lane >> 4;
    return 2 * S::at(4 * (grp >> 1) + (s >> 2), 16 * (grp & 1) + 4 * (s & 3));
  }
  static __device__ __forceinline__ unsigned col_block(unsigned cols, int m) { return cols ^ (64 * m); }  // by_col's m counts from there
  static __device__ __forceinline__ Frag8<bf16_t> by_col(unsigned cols, int off, int m) {
    typedef short short4_ __attribute__((ext_vector_type(4)));
    typedef short short8_ __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) short4_ lds_short4;
    // eight rows further on x differs by 2 in its low bits (128-byte and 256-byte rows alike)
    const unsigned at = cols ^ (64 * m);
    const short4_ lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds_char*)(uintptr_t)(at + off));
    const short4_ hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds_char*)(uintptr_t)((at ^ 32) + off + 8 * ROWB));
    const short8_ v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return {__builtin_bit_cast(bf16x8, v)};
  }
};
template <int D, int R> struct Tile<float, D, R> {
  static constexpr int BYTES = R * D * 4, ROWB = D * 4, G = D / 4;
  static __device__ __forceinline__ int at(int r, int c) { return r * D + ((((c >> 2) ^ (r & 7)) << 2) | (c & 3)); }
  static __device__ __forceinline__ void src(int j, int lane, int& r, int& c) {
    const int p = 64 * j + lane;
    r = p / G;
    c = ((p % G) ^ (r & 7)) << 2;
  }
  static __device__ __forceinline__ unsigned rows(int lane) { return 4 * at(lane & 31, 8 * (lane >> 5)); }
  static __device__ __forceinline__ Frag8<float> by_row(unsigned rows, int off, int s) {
    const floatx4 a = lds_load<floatx4>((rows ^ (64 * s)) + off), b = lds_load<floatx4>((rows ^ (64 * s + 16)) + off);
    return {{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]}};
  }
  static __device__ __forceinline__ unsigned cols(int lane) { return 4 * at(4 * (lane >> 5), lane & 31); }
  static __device__ __forceinline__ unsigned col_block(unsigned cols, int m) { return cols + 128 * m; }
  static __device__ __forceinline__ Frag8<float> by_col(unsigned cols, int off, int m) {
    Frag8<float> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f.v[e] = lds_load<float>((cols ^ (16 * (e & 3))) + off + (8 * (e >> 2) + (e & 3)) * ROWB + 128 * m);
    return f;
  }
};

// 16 bytes a lane from `base` + off bytes straight to LDS, lane l at dst + 16 l; the base is the wave's, so a tile's loads cost no
// vector arithmetic
__device__ __forceinline__ void dma16_at(const void* base, unsigned off, unsigned dst) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(__builtin_amdgcn_readfirstlane(dst)) : "memory", "m0");
}
// Brings tiles of [len][d] matrices with one row stride to LDS by the workgroup's four waves: which bytes a lane fetches is formed once.
template <typename T, int D, int R = ROWS> struct Mover {
  typedef Tile<T, D, R> TL;
  static constexpr int N = TL::BYTES / 1024 / 4;
  unsigned off[N];
  int64_t st;
  int d, lane, wave;
  __device__ __forceinline__ Mover(int64_t st_, int d_, int wave_, int lane_) : st(st_), d(d_), lane(lane_), wave(wave_) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int r, c;
      TL::src(wave * N + i, lane, r, c);
      off[i] = (unsigned)((r * (int)st + c) * (int)sizeof(T));
    }
  }
  // rows row0 .. row0 + R - 1; rows behind the last are copies of the last, columns behind d keep the zeros that clear_lds left
  __device__ __forceinline__ void fetch(unsigned tile, const T* matrix, int row0, int len) const {
    if (row0 + R <= len && d == D) {
      const T* base = matrix + (int64_t)row0 * st;
#pragma unroll
      for (int i = 0; i < N; ++i) dma16_at(base, off[i], tile + 1024 * (wave * N + i));
    } else {
#pragma unroll 1
      for (int i = 0; i < N; ++i) {
        int r, c;
        TL::src(wave * N + i, lane, r, c);
        if (c < d) dma16(matrix + (int64_t)min(row0 + r, len - 1) * st + c, tile + 1024 * (wave * N + i));
      }
    }
  }
};
__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }
// What the rounding of that operand left, as a second operand.  WEIGHTS: the values are at most 2^8 or NaN (of a score gradient that is
// infinite, or becomes so, nothing is left).
template <bool WEIGHTS> __device__ __forceinline__ void rest_of(Frag8<bf16_t>& f, const floatx16& c, int h, const Frag8<bf16_t>& rounded) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f.v[e] = from_f32<bf16_t>(WEIGHTS || is_finite(to_f32(rounded.v[e])) ? c[8 * h + e] - to_f32(rounded.v[e]) : 0.f);
}
template <bool WEIGHTS> __device__ __forceinline__ void rest_of(Frag8<float>&, const floatx16&, int, const Frag8<float>&) {}
// Whether the granules that this lane's loads brought hold finite values only; SCRUB: the others become 0.  A wave's granules are
// the rows of its quarter of the tile.
template <typename T, int D, bool SCRUB, int R = ROWS> __device__ __forceinline__ bool tile_finite(T* tile, int wave, int lane) {
  constexpr int N = Tile<T, D, R>::BYTES / 1024 / 4, VN = Vec16<T>::N;
  bool ok = true;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    typename Vec16<T>::V* p = reinterpret_cast<typename Vec16<T>::V*>(tile + (64 * (wave * N + i) + lane) * VN);
    typename Vec16<T>::V v = *p;
    bool all = true;
#pragma unroll
    for (int e = 0; e < VN; ++e)
      if (!is_finite(to_f32(v[e]))) all = false, v[e] = from_f32<T>(0.f);
    if (SCRUB && !all) *p = v;
    ok = ok && all;
  }
  return ok;
}
__device__ __forceinline__ void clear_lds(char* p, int bytes) {
  for (int i = threadIdx.x * 16; i < bytes; i += 256 * 16) *reinterpret_cast<floatx4*>(p + i) = floatx4{0.f, 0.f, 0.f, 0.f};
}

// How a run of N products takes its operands from LDS (COL: through by_col): AHEAD operands are on their way before the first product
// and each product is followed by the reads of another.  Left to itself the compiler saves the registers and waits for every operand
// right before its product, 130 cycles for 32 of work.  EACH: products that take the same operand.
template <typename T, bool COL, int N, int AHEAD, int EACH = 1> __device__ __forceinline__ void read_ahead() {
  constexpr int READS = sizeof(T) == 2 ? (COL ? 2 : 1) : (COL ? 8 : 2), PRODUCTS = EACH * (sizeof(T) == 2 ? 1 : 8), DS = 0x100, MFMA = 0x8;
  __builtin_amdgcn_sched_group_barrier(DS, READS * AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N - AHEAD; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, PRODUCTS, 0);
    __builtin_amdgcn_sched_group_barrier(DS, READS, 0);
  }
  __builtin_amdgcn_sched_group_barrier(MFMA, PRODUCTS * AHEAD, 0);
}

// max over the wave's two halves
__device__ __forceinline__ float half_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// A product over the rows of a tile takes masked pairs with weight 0, and 0 times a value that is not finite is not 0: such values
// are scrubbed from the tile, and their part of the product is added here, pair by pair and only where keep(row) lets this lane's
// column have it.  w: the weights of the 32 rows from row0 on, as an operand; the values are read again from memory.
template <typename T, int M, typename F>
__device__ __forceinline__ void add_odd(floatx16 (&acc)[M], const T* base, int64_t st, int row0, int len, int d, const Frag8<T> (&w)[2], int lane, F keep) {
  const int kg = lane >> 5;
#pragma unroll 1
  for (int j = 0; j < 32 && row0 + j < len; ++j) {
    const int e = (j & 3) + 4 * (j >> 3);
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) x = e == i ? to_f32(w[i >> 3].v[i & 7]) : x;
    const float other = __shfl_xor(x, 32, LNX_WAVE);
    x = ((j >> 2) & 1) == kg ? x : other;
    const bool on = keep(row0 + j);
    const T* r = base + (int64_t)(row0 + j) * st + 4 * kg;
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (32 * m + 8 * q + 4 * kg < d) {
          const floatx4 v = load4(r + 32 * m + 8 * q);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (on && !is_finite(v[i])) acc[m][4 * q + i] += x * v[i];
        }
  }
}

// Where a workgroup works: sequence (its first token, its length), block of `size` rows, heads
struct Place {
  int b, hkv, g, part, len, blk;
  int64_t tok;
  bool on;
};
// `heads`: query heads of a group that have workgroups of their own -- all or one; each block is split into a.parts.  Heavy blocks first: of causal queries
// the last ones (`last_first`), of keys the first ones.  Where the groups divide among the eight XCDs, workgroups of one group stay on
// one, whose L2 then holds the group's keys and values.
__device__ __forceinline__ Place place(const Args& a, int size, int heads, bool last_first) {
  Place p;
  int w = blockIdx.x, group, blk;
  const int groups = a.B * a.Hkv, per_group = heads * a.parts;
  if (groups % 8 == 0) {
    const int slot = w >> 3, here = groups / 8 * per_group;
    blk = slot / here;
    w = slot % here;
    group = (w / per_group) * 8 + (blockIdx.x & 7);
    w %= per_group;
  } else {
    blk = w / (groups * per_group);
    w -= blk * groups * per_group;
    group = w / per_group;
    w %= per_group;
  }
  p.g = w / a.parts;
  p.part = w % a.parts;
  p.b = group / a.Hkv;
  p.hkv = group % a.Hkv;
  p.tok = 0;
  p.len = a.T;
  p.on = true;
  if (!a.nseq) {
    p.blk = last_first ? a.nblk - 1 - blk : blk;
    return p;
  }
  const int seq = packed_owner(a.cu, a.nseq, a.T, size, blk);
  p.tok = seq_first(a.cu, seq, a.T);
  p.len = seq_end(a.cu, seq, a.T) - (int)p.tok;
  const int n = (int)(((unsigned)p.len + size - 1) / size);
  p.blk = (int)(blk - packed_slot((int)p.tok, seq, size));
  p.on = p.blk >= 0 && p.blk < n;
  if (last_first) p.blk = n - 1 - p.blk;
  return p;
}
template <typename T> __device__ __forceinline__ T* at(const void* p, const int64_t (&s)[3], int64_t b, int64_t h, int64_t t) {
  return const_cast<T*>(static_cast<const T*>(p)) + b * s[0] + h * s[1] + t * s[2];
}

// One column's 32 M values from accumulators over rows, the first d of them, times f: the lane writes four consecutive elements at a time
template <typename T, int M> __device__ __forceinline__ void store_column(T* p, const floatx16 (&acc)[M], float f, int d, int lane) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * m + 8 * q + 4 * (lane >> 5);
      if (c < d) store4(p + c, floatx4{acc[m][4 * q] * f, acc[m][4 * q + 1] * f, acc[m][4 * q + 2] * f, acc[m][4 * q + 3] * f});
    }
}

// What the rounding of such a column left
template <typename T, int M> __device__ __forceinline__ void store_low(T* p, const floatx16 (&acc)[M], float f, int d, int lane) {
#pragma unroll
  for (int m = 0; m < M; ++m)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = 32 * m + 8 * q + 4 * (lane >> 5);
      floatx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = acc[m][4 * q + e] * f;
        v[e] = x - to_f32(from_f32<T>(x));
      }
      if (c < d) store4(p + c, v);
    }
}

// Keys of a tile of the forward pass: with 32 three workgroups share a CU (registers, LDS) and less of the diagonal is wasted: eight packed
// prompts of 8192 tokens together 175 us with 64, 160 with 32; B2 H16/4 T4096 154 and 156.
template <typename T, int D> constexpr int fwd_rows() { return sizeof(T) == 2 && D == 128 ? 32 : 64; }

// TWO (all three kernels): weights and score gradients enter the products in two bf16 parts.  For sequences of up to SHORT tokens: a
// gradient there is a sum of a few terms, whose roundings (2^-8 each) do not average out: of three tokens dq and dk were 1.8 times as
// far off as their own rounding leaves them, of 64 and more 1.4 times.  Every workgroup goes by its own sequence, so that a document's
// operands do not depend on what it is packed with; kernels that may meet both kinds hold both forms (MIXED: packed batches; forward of
// eight prompts of 8192 tokens together 161 us with one form, 163 with both, backward 623 and 636).  128 tokens are one block of queries.  By the average
// length a document of 8000 tokens among 150 of one, H16/4 d128, took 422 us forward and 2035 backward, this way 305 and 1405; 2048 of
// 128, H8/2 d128, in one part 760 and 1955, in two 759 and 2247.
constexpr int SHORT = 128;

// A wave owns 32 queries, the workgroup 128; of a block's key tiles every a.parts-th.
template <typename T, int D, bool TWO> __device__ __forceinline__ void fwd_block(const Args& a, const Place& p, char* lds) {
  constexpr int KT = fwd_rows<T, D>(), KH = KT / 32;
  typedef Tile<T, D, KT> TL;
  const auto kt = [=](int buf) { return reinterpret_cast<T*>(lds + 2 * buf * TL::BYTES); };
  const auto vt = [=](int buf) { return reinterpret_cast<T*>(lds + (2 * buf + 1) * TL::BYTES); };
  int* odd = reinterpret_cast<int*>(lds + 4 * TL::BYTES);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, kg = lane >> 5;
  const int h = p.hkv * a.G + p.g, q_wg = p.blk * 128, q0 = q_wg + wave * 32, q = q0 + n;
  const T* kb = at<T>(a.k, a.ks, p.b, p.hkv, p.tok);
  const T* vb = at<T>(a.v, a.vs, p.b, p.hkv, p.tok);
  const int q_end = min(q_wg + 128, p.len), ntile = (q_end + KT - 1) / KT;
  if (a.d < D) clear_lds(lds, 4 * TL::BYTES);
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;
  lds_barrier();
  const Mover<T, D, KT> mk(a.ks[2], a.d, wave, lane), mv(a.vs[2], a.d, wave, lane);
  const unsigned lds0 = lds_byte_addr(lds);
  if (p.part < ntile) {
    mk.fetch(lds0, kb, p.part * KT, p.len);
    mv.fetch(lds0 + TL::BYTES, vb, p.part * KT, p.len);
  }
  // queries as B operands; a negative scale turns their sign, so that the largest product has the largest score
  const float c = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f);  // above 0: -inf stays what a masked score is
  Frag8<T> qf[D / 16];
  const T* qr = at<T>(a.q, a.qs, p.b, h, p.tok + min(q, p.len - 1));
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    from_global<T>(qf[s], qr + 16 * s + 8 * kg, 16 * s + 8 * kg < a.d);
    if (a.scale < 0.f)
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[s].v[e] = -qf[s].v[e];
  }
  floatx16 acc[D / 32];
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  const unsigned row_addr = lds0 + TL::rows(lane), col_addr = lds0 + TL::cols(lane);
  for (int it = p.part, buf = 0; it < ntile; it += a.parts, buf ^= 1) {
    const int key0 = it * KT, next = key0 + a.parts * KT;
    const unsigned rows = row_addr + 2 * buf * TL::BYTES, cols = col_addr + 2 * buf * TL::BYTES;
    dma_wait<0>();
    const bool edge = key0 + KT > q_wg;  // some pairs of this tile are masked
    if (edge && !tile_finite<T, D, true, KT>(vt(buf), wave, lane)) odd[buf] = 1;
    lds_barrier();
    if (it + a.parts < ntile) {
      mk.fetch(lds0 + 2 * (buf ^ 1) * TL::BYTES, kb, next, p.len);
      mv.fetch(lds0 + (2 * (buf ^ 1) + 1) * TL::BYTES, vb, next, p.len);
    }
    if (key0 >= q0 + 32) continue;  // behind all of this wave's queries
    floatx16 sc[KH];
#pragma unroll
    for (int i = 0; i < KH; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[i][e] = 0.f;
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int i = 0; i < KH; ++i)
#pragma unroll
      for (int s = 0; s < D / 16; ++s) mma(sc[i], TL::by_row(rows, 32 * i * TL::ROWB, s), qf[s]);
    read_ahead<T, false, KH * (D / 16), 4>();
    __builtin_amdgcn_s_setprio(0);
    if (key0 + KT - 1 > q0) {
#pragma unroll
      for (int i = 0; i < KH; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + 32 * i + frag_row(e, lane) > q) sc[i][e] = -INFINITY;
    }
    float top = sc[0][0];
#pragma unroll
    for (int i = 0; i < KH; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, sc[i][e]);
    top = half_max(top);
    // a new reference only where the old one is short by more than 2^8: sums and accumulators stay far inside fp32's range
    if (__any(top > m + 8.f / c || (m == -INFINITY && top > m))) {
      const float higher = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - higher) * c);
      l *= f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] *= f;
      m = higher;
    }
    const float ref = m == -INFINITY ? 0.f : m * c;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < KH; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sc[i][e] = __builtin_amdgcn_exp2f(sc[i][e] * c - ref);
        sum += sc[i][e];
      }
    l += sum;
    Frag8<T> pf[2 * KH], rest[2 * KH];
#pragma unroll
    for (int s = 0; s < 2 * KH; ++s) {
      from_acc(pf[s], sc[s >> 1], s & 1);
      if constexpr (TWO) rest_of<true>(rest[s], sc[s >> 1], s & 1, pf[s]);
    }
#pragma unroll
    for (int s = 0; s < 2 * KH; ++s)
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const Frag8<T> v = TL::by_col(cols, TL::BYTES + 16 * s * TL::ROWB, i);
        mma(acc[i], v, pf[s]);
        if constexpr (TWO) mma(acc[i], v, rest[s]);
      }
    read_ahead<T, true, 2 * KH * (D / 32), TWO ? 1 : 4, TWO ? 2 : 1>();  // (four ahead of two products each spill: 1134 us for those 2048, 759)
    if (edge && odd[buf])
#pragma unroll
      for (int i = 0; i < KH; ++i) {
        const Frag8<T> two[2] = {pf[2 * i], pf[2 * i + 1]};
        add_odd<T, D / 32>(acc, vb, a.vs[2], key0 + 32 * i, p.len, a.d, two, lane, [&](int row) { return row <= q; });
      }
  }
  const float sum = xor32_sum(l);
  if (q >= p.len) return;
  const int64_t row = ((int64_t)p.b * a.H + h) * a.T + p.tok + q;
  if (a.parts == 1) {
    store_column<T, D / 32>(at<T>(a.o, a.os, p.b, h, p.tok + q), acc, 1.f / sum, a.d, lane);
    if (a.o_low) store_low<T, D / 32>(static_cast<T*>(a.o_low) + row * a.d, acc, 1.f / sum, a.d, lane);
    if (a.lse && kg == 0) a.lse[row] = m * c + __builtin_amdgcn_logf(sum);
  } else {
    const int64_t at_part = (int64_t)p.part * a.B * a.H * a.T + row;
    store_column<float, D / 32>(a.part + at_part * a.d, acc, 1.f, a.d, lane);
    if (kg == 0) a.part_stat[2 * at_part] = m * c, a.part_stat[2 * at_part + 1] = sum;
  }
}

template <typename T, int D, bool MIXED> __global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : 3) void attn_fwd_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Place p = place(a, 128, a.G, true);
  if (!p.on) return;
  if (MIXED && __builtin_amdgcn_readfirstlane(p.len) <= SHORT) fwd_block<T, D, MIXED>(a, p, lds);
  else fwd_block<T, D, false>(a, p, lds);
}

// The parts of a row's result, sixteen lanes a row
template <typename T> __global__ __launch_bounds__(256) void attn_join_kernel(Args a) {
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), all = (int64_t)a.B * a.H * a.T;
  const int c = 8 * (threadIdx.x & 15);
  if (row >= all || c >= a.d) return;
  float top = -INFINITY, sum = 0.f, o[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] = 0.f;
  for (int s = 0; s < a.parts; ++s) top = fmaxf(top, a.part_stat[2 * (s * all + row)]);
  for (int s = 0; s < a.parts; ++s) {
    const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(a.part_stat[2 * (s * all + row)] - top);
    sum += a.part_stat[2 * (s * all + row) + 1] * f;
    const float* p = a.part + (s * all + row) * a.d + c;
    const floatx4 x = load4(p), y = load4(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += x[e] * f, o[e + 4] += y[e] * f;
  }
  const int64_t t = row % a.T, bh = row / a.T;
  T* p = at<T>(a.o, a.os, bh / a.H, bh % a.H, t) + c;
#pragma unroll
  for (int e = 0; e < 8; ++e) o[e] /= sum;
  store4(p, floatx4{o[0], o[1], o[2], o[3]});
  store4(p + 4, floatx4{o[4], o[5], o[6], o[7]});
  if (a.o_low) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] -= to_f32(from_f32<T>(o[e]));
    T* low = static_cast<T*>(a.o_low) + row * a.d + c;
    store4(low, floatx4{o[0], o[1], o[2], o[3]});
    store4(low + 4, floatx4{o[4], o[5], o[6], o[7]});
  }
  if (a.lse && c == 0) a.lse[row] = top + __builtin_amdgcn_logf(sum);
}

// The sum of the parts [parts][stride rows][d] of a [B, heads, T, d] gradient, sixteen lanes a row
template <typename T> __global__ __launch_bounds__(256) void attn_sum_kernel(const float* part, int parts, int64_t stride, T* out, int64_t sb, int64_t sh, int64_t st, int B,
                                                                             int heads, int T_, int d) {
  const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int c = 8 * (threadIdx.x & 15);
  if (row >= (int64_t)B * heads * T_ || c >= d) return;
  floatx4 x = {0.f, 0.f, 0.f, 0.f}, y = x;
  for (int s = 0; s < parts; ++s) {
    const float* p = part + (s * stride + row) * d + c;
    x += load4(p);
    y += load4(p + 4);
  }
  const int64_t t = row % T_, bh = row / T_;
  T* p = out + bh / heads * sb + bh % heads * sh + t * st + c;
  store4(p, x);
  store4(p + 4, y);
}

// Queries as in the forward pass, their gradients beside them in registers.  delta is formed here, for the dk / dv kernel too: of o and
// what its rounding left, because an error of delta goes into every term of a row of dq (rounded o alone: 1.5 times the error that the
// rounding of dq has, with it 1.4).
template <typename T, int D, bool TWO> __device__ __forceinline__ void dq_block(const Args& a, const Place& p, char* lds) {
  typedef Tile<T, D> TL;
  const auto kt = [=](int buf) { return reinterpret_cast<T*>(lds + 2 * buf * TL::BYTES); };
  int* odd = reinterpret_cast<int*>(lds + 4 * TL::BYTES);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, kg = lane >> 5;
  const int h = p.hkv * a.G + p.g, q_wg = p.blk * 128, q0 = q_wg + wave * 32, q = q0 + n;
  const T* kb = at<T>(a.k, a.ks, p.b, p.hkv, p.tok);
  const T* vb = at<T>(a.v, a.vs, p.b, p.hkv, p.tok);
  const int q_end = min(q_wg + 128, p.len), ntile = (q_end + ROWS - 1) / ROWS;
  if (a.d < D) clear_lds(lds, 4 * TL::BYTES);
  if (threadIdx.x < 2) odd[threadIdx.x] = 0;
  lds_barrier();
  const Mover<T, D> mk(a.ks[2], a.d, wave, lane), mv(a.vs[2], a.d, wave, lane);
  const unsigned lds0 = lds_byte_addr(lds);
  if (p.part < ntile) {
    mk.fetch(lds0, kb, p.part * ROWS, p.len);
    mv.fetch(lds0 + TL::BYTES, vb, p.part * ROWS, p.len);
  }
  const float c = a.scale * LOG2E;
  const int64_t row = min(q, p.len - 1), stat = ((int64_t)p.b * a.H + h) * a.T + p.tok + row;
  const float lse = a.lse[stat];
  const T* qr = at<T>(a.q, a.qs, p.b, h, p.tok + row);
  const T* gr = at<T>(a.dout, a.gs, p.b, h, p.tok + row);
  const T* orow = at<T>(a.o, a.os, p.b, h, p.tok + row);
  const T* lrow = a.o_low ? static_cast<const T*>(a.o_low) + stat * a.d : nullptr;
  Frag8<T> qf[D / 16], gf[D / 16];
  float delta = 0.f;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    const int at = 16 * s + 8 * kg;
    from_global<T>(qf[s], qr + at, at < a.d);
    from_global<T>(gf[s], gr + at, at < a.d);
    Frag8<T> o, low;
    from_global<T>(o, orow + at, at < a.d);
    from_global<T>(low, lrow + at, lrow && at < a.d);
#pragma unroll
    for (int e = 0; e < 8; ++e) delta += (to_f32(o.v[e]) + to_f32(low.v[e])) * to_f32(gf[s].v[e]);
  }
  delta = xor32_sum(delta);
  if (kg == 0 && q < p.len) a.delta[stat] = delta;  // every part writes the same
  floatx16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  const unsigned row_addr = lds0 + TL::rows(lane), col_addr = lds0 + TL::cols(lane);
  for (int it = p.part, buf = 0; it < ntile; it += a.parts, buf ^= 1) {
    const int key0 = it * ROWS, next = key0 + a.parts * ROWS;
    const unsigned rows = row_addr + 2 * buf * TL::BYTES, cols = col_addr + 2 * buf * TL::BYTES;
    dma_wait<0>();
    const bool edge = key0 + ROWS > q_wg;
    if (edge && !tile_finite<T, D, false>(kt(buf), wave, lane)) odd[buf] = 1;
    lds_barrier();
    if (it + a.parts < ntile) {
      mk.fetch(lds0 + 2 * (buf ^ 1) * TL::BYTES, kb, next, p.len);
      mv.fetch(lds0 + (2 * (buf ^ 1) + 1) * TL::BYTES, vb, next, p.len);
    }
    const bool scrub = edge && odd[buf];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool mine = key0 + 32 * i <= q0 + 31;  // not behind all of this wave's queries
      Frag8<T> ds[2], rest[2];
      if (mine) {
        floatx16 sc, dp;
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = dp[e] = 0.f;
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
          mma(sc, TL::by_row(rows, 32 * i * TL::ROWB, s), qf[s]);
          mma(dp, TL::by_row(rows, TL::BYTES + 32 * i * TL::ROWB, s), gf[s]);
        }
        read_ahead<T, false, 2 * (D / 16), 4>();
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int e = 0; e < 16; ++e) sc[e] = __builtin_amdgcn_exp2f(sc[e] * c - lse) * (dp[e] - delta);
        if (key0 + 32 * i + 31 > q0)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            if (key0 + 32 * i + frag_row(e, lane) > q) sc[e] = 0.f;
        from_acc(ds[0], sc, 0);
        from_acc(ds[1], sc, 1);
        if constexpr (TWO) rest_of<false>(rest[0], sc, 0, ds[0]), rest_of<false>(rest[1], sc, 1, ds[1]);
      }
      if (scrub) {  // the scores are made of the keys as they are
        lds_barrier();
        if (wave >> 1 == i) tile_finite<T, D, true>(kt(buf), wave, lane);
        lds_barrier();
      }
      if (mine) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int m = 0; m < D / 32; ++m) {
            const Frag8<T> k = TL::by_col(cols, (32 * i + 16 * s) * TL::ROWB, m);
            mma(acc[m], k, ds[s]);
            if constexpr (TWO) mma(acc[m], k, rest[s]);
          }
        read_ahead<T, true, 2 * (D / 32), 4, TWO ? 2 : 1>();
        if (scrub) add_odd<T, D / 32>(acc, kb, a.ks[2], key0 + 32 * i, p.len, a.d, ds, lane, [&](int row) { return row <= q; });
      }
    }
  }
  if (q >= p.len) return;
  if (a.parts == 1) store_column<T, D / 32>(at<T>(a.dq, a.dqs, p.b, h, p.tok + q), acc, a.scale, a.d, lane);
  else store_column<float, D / 32>(a.part + ((int64_t)p.part * a.B * a.H * a.T + stat) * a.d, acc, a.scale, a.d, lane);
}

template <typename T, int D, bool MIXED> __global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_dq_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Place p = place(a, 128, a.G, true);
  if (!p.on) return;
  if (MIXED && __builtin_amdgcn_readfirstlane(p.len) <= SHORT) dq_block<T, D, MIXED>(a, p, lds);
  else dq_block<T, D, false>(a, p, lds);
}

// An operand through LDS to another wave of the workgroup
template <typename T> __device__ __forceinline__ void leave_frag(unsigned at, const Frag8<T>& f, int lane) {
  typedef __attribute__((address_space(3))) floatx4 lds_float4;
  const floatx4* v = reinterpret_cast<const floatx4*>(&f);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) *(lds_float4*)(lds_char*)(uintptr_t)(at + 1024 * i + 16 * lane) = v[i];
}
template <typename T> __device__ __forceinline__ void take_frag(unsigned at, Frag8<T>& f, int lane) {
  floatx4* v = reinterpret_cast<floatx4*>(&f);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = lds_load<floatx4>(at + 1024 * i + 16 * lane);
}

template <typename T> constexpr int hand_over() { return 8192 * (int)sizeof(T); }  // bytes of a workgroup

// A workgroup owns 64 keys.  Wave (kw, qw) forms the weights of 32 keys and the half qw of a tile's queries, hands them to the wave of
// the other half, and adds up the half qw of the columns of dk and dv over all queries: accumulators of half the size, so that two
// workgroups share a CU.  (With both halves in every wave it took 416 registers and one workgroup a CU; as long, 456 and 469 us at B2 H16/4
// T4096 d128, while the first keys' workgroups, which walk over all queries, were what the launch waited for.  Their queries split into
// parts need the second workgroup: 317 us.)  The LDS of a workgroup is 80 KB to the byte: the queries' lse and delta go straight to
// registers, a flag crosses in the hand-over's place.  In two parts twice as much is handed over, in the place of the second buffer of
// tiles, and the next tile is fetched when the waves have done with the one before: a short sequence has one or two for each query head.
template <typename T, int D, bool TWO> __device__ __forceinline__ void dkv_block(const Args& a, const Place& p, char* lds) {
  typedef Tile<T, D> TL;
  typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
  constexpr int M = D / 64, FRAG = 1024 * (int)sizeof(T) / 2, HAND = hand_over<T>() / 4 * (TWO ? 2 : 1);  // bytes that a wave hands over
  constexpr int BUFS = TWO ? 1 : 2;
  static_assert(2 * BUFS * TL::BYTES + 4 * HAND <= 4 * TL::BYTES + hand_over<T>(), "both forms have the same LDS");
  const auto qt = [=](int buf) { return reinterpret_cast<T*>(lds + 2 * buf * TL::BYTES); };
  const auto gt = [=](int buf) { return reinterpret_cast<T*>(lds + (2 * buf + 1) * TL::BYTES); };
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, kg = lane >> 5;
  const int kw = wave & 1, qw = wave >> 1, r0 = 32 * qw, key0 = p.blk * ROWS + 32 * kw, key = key0 + n;
  const int per = (p.len + ROWS - 1) / ROWS - p.blk, total = per * a.G, last = (p.blk + per) * ROWS;
  if (a.d < D) {
    clear_lds(lds, 4 * TL::BYTES);
    lds_barrier();
  }
  const Mover<T, D> mq(a.qs[2], a.d, wave, lane), mg(a.gs[2], a.d, wave, lane);
  const unsigned lds0 = lds_byte_addr(lds), hand = lds0 + 2 * BUFS * TL::BYTES, mine = hand + HAND * wave, theirs = hand + HAND * (wave ^ 2);
  floatx4 lse[4], delta[4];
  auto fetch_stats = [&](int h, int row0) {
    const int64_t first = ((int64_t)p.b * a.H + h) * a.T + p.tok;
    const int row = row0 + r0 + 4 * kg;
    if (row0 + ROWS <= p.len) {
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        lse[g] = *reinterpret_cast<const float4u*>(a.lse + first + row + 8 * g);
        delta[g] = *reinterpret_cast<const float4u*>(a.delta + first + row + 8 * g);
      }
    } else {
#pragma unroll
      for (int g = 0; g < 4; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int64_t at = first + min(row + 8 * g + e, p.len - 1);
          lse[g][e] = a.lse[at];
          delta[g][e] = a.delta[at];
        }
    }
  };
  auto fetch = [&](int h, int row0, int buf) {
    mq.fetch(lds0 + 2 * buf * TL::BYTES, at<T>(a.q, a.qs, p.b, h, p.tok), row0, p.len);
    mg.fetch(lds0 + (2 * buf + 1) * TL::BYTES, at<T>(a.dout, a.gs, p.b, h, p.tok), row0, p.len);
  };
  // of the (query head, tile of queries) pairs every a.parts-th: the one being multiplied
  int h = p.hkv * a.G + p.part / per, row0 = (p.blk + p.part % per) * ROWS;
  if (p.part < total) {
    fetch(h, row0, 0);
    fetch_stats(h, row0);
  }
  const float c = a.scale * LOG2E;
  const int64_t krow = p.tok + min(key, p.len - 1);
  const T* kr = at<T>(a.k, a.ks, p.b, p.hkv, krow);
  const T* vr = at<T>(a.v, a.vs, p.b, p.hkv, krow);
  Frag8<T> kf[D / 16], vf[D / 16];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    from_global<T>(kf[s], kr + 16 * s + 8 * kg, 16 * s + 8 * kg < a.d);
    from_global<T>(vf[s], vr + 16 * s + 8 * kg, 16 * s + 8 * kg < a.d);
  }
  floatx16 dk[M], dv[M];
#pragma unroll
  for (int i = 0; i < M; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) dk[i][e] = dv[i][e] = 0.f;
  const unsigned row_addr = lds0 + r0 * TL::ROWB + TL::rows(lane), col_addr = TL::col_block(lds0 + TL::cols(lane), M * qw);
  for (int it = p.part, buf = 0; it < total; it += a.parts, buf ^= BUFS - 1) {
    dma_wait<0>();
#pragma unroll
    for (int g = 0; g < 4; ++g) asm volatile("" : "+v"(lse[g]), "+v"(delta[g]));  // have come too: no wait for the next tile at their use
    const bool edge = row0 == p.blk * ROWS || row0 + ROWS > p.len;
    int next_h = h, next_row0 = row0 + a.parts * ROWS;
    for (; next_row0 >= last; ++next_h) next_row0 -= per * ROWS;
    lds_barrier();
    bool scrub = false;
    if (edge) {
      const bool ok = tile_finite<T, D, false>(qt(buf), wave, lane) && tile_finite<T, D, false>(gt(buf), wave, lane);
      typedef __attribute__((address_space(3))) int lds_int;
      const int all = __all(ok);
      if (lane == 0) *(lds_int*)(lds_char*)(uintptr_t)mine = !all;
      lds_barrier();
#pragma unroll
      for (int w = 0; w < 4; ++w) scrub = scrub || lds_load<int>(hand + HAND * w) != 0;
      scrub = __builtin_amdgcn_readfirstlane(scrub);
      lds_barrier();
    }
    if (!TWO && it + a.parts < total) fetch(next_h, next_row0, buf ^ 1);
    const unsigned rows = row_addr + 2 * buf * TL::BYTES, cols = col_addr + 2 * buf * TL::BYTES;
    const auto active = [&](int q) { return row0 + 32 * q + 31 >= key0 && row0 + 32 * q < p.len; };  // some of these queries come after some of the keys
    Frag8<T> pf[2], ds[2];
    if (active(qw)) {
      floatx16 sc, dp;
#pragma unroll
      for (int e = 0; e < 16; ++e) sc[e] = dp[e] = 0.f;
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) mma(sc, TL::by_row(rows, 0, s), kf[s]);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) mma(dp, TL::by_row(rows, TL::BYTES, s), vf[s]);
      read_ahead<T, false, 2 * (D / 16), 4>();
      __builtin_amdgcn_s_setprio(0);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        sc[e] = __builtin_amdgcn_exp2f(sc[e] * c - lse[e >> 2][e & 3]);
        dp[e] = sc[e] * (dp[e] - delta[e >> 2][e & 3]);
      }
      if (edge)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int q = row0 + r0 + frag_row(e, lane);
          if (q < key || q >= p.len) sc[e] = dp[e] = 0.f;
        }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        from_acc(pf[s], sc, s);
        from_acc(ds[s], dp, s);
        leave_frag<T>(mine + s * FRAG, pf[s], lane);
        leave_frag<T>(mine + (2 + s) * FRAG, ds[s], lane);
        if constexpr (TWO) {
          Frag8<T> rest;
          rest_of<true>(rest, sc, s, pf[s]);
          leave_frag<T>(mine + (4 + s) * FRAG, rest, lane);
          rest_of<false>(rest, dp, s, ds[s]);
          leave_frag<T>(mine + (6 + s) * FRAG, rest, lane);
        }
      }
    }
    if (it + a.parts < total) fetch_stats(next_h, next_row0);
    lds_barrier();
    if (scrub) {  // the scores were made of the queries and gradients as they are
      tile_finite<T, D, true>(qt(buf), wave, lane);
      tile_finite<T, D, true>(gt(buf), wave, lane);
      lds_barrier();
    }
    const auto add = [&](int half, unsigned area) {
      const unsigned from = cols + 32 * half * TL::ROWB;
      Frag8<T> pr[2], dr[2];
      if constexpr (TWO)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          take_frag<T>(area + (4 + s) * FRAG, pr[s], lane);
          take_frag<T>(area + (6 + s) * FRAG, dr[s], lane);
        }
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int m = 0; m < M; ++m) {
          const Frag8<T> g = TL::by_col(from, TL::BYTES + 16 * s * TL::ROWB, m);
          mma(dv[m], g, pf[s]);
          if constexpr (TWO) mma(dv[m], g, pr[s]);
          const Frag8<T> q = TL::by_col(from, 16 * s * TL::ROWB, m);
          mma(dk[m], q, ds[s]);
          if constexpr (TWO) mma(dk[m], q, dr[s]);
        }
      read_ahead<T, true, 4 * M, 4, TWO ? 2 : 1>();
      if (scrub) {
        const auto keep = [&](int row) { return row >= key; };
        add_odd<T, M>(dv, at<T>(a.dout, a.gs, p.b, h, p.tok) + 32 * M * qw, a.gs[2], row0 + 32 * half, p.len, a.d - 32 * M * qw, pf, lane, keep);
        add_odd<T, M>(dk, at<T>(a.q, a.qs, p.b, h, p.tok) + 32 * M * qw, a.qs[2], row0 + 32 * half, p.len, a.d - 32 * M * qw, ds, lane, keep);
      }
    };
    if (active(qw)) add(qw, mine);
    if (active(qw ^ 1)) {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        take_frag<T>(theirs + s * FRAG, pf[s], lane);
        take_frag<T>(theirs + (2 + s) * FRAG, ds[s], lane);
      }
      add(qw ^ 1, theirs);
    }
    if (TWO && it + a.parts < total) {
      lds_barrier();
      fetch(next_h, next_row0, 0);
    }
    h = next_h;
    row0 = next_row0;
  }
  if (key >= p.len) return;
  const int c0 = 32 * M * qw;
  if (a.parts == 1) {
    store_column<T, M>(at<T>(a.dk, a.dks, p.b, p.hkv, krow) + c0, dk, a.scale, a.d - c0, lane);
    store_column<T, M>(at<T>(a.dv, a.dvs, p.b, p.hkv, krow) + c0, dv, 1.f, a.d - c0, lane);
  } else {
    const int64_t rows_all = (int64_t)a.B * a.Hkv * a.T, at_part = 2 * p.part * rows_all + ((int64_t)p.b * a.Hkv + p.hkv) * a.T + krow;
    store_column<float, M>(a.part + at_part * a.d + c0, dk, a.scale, a.d - c0, lane);
    store_column<float, M>(a.part + (at_part + rows_all) * a.d + c0, dv, 1.f, a.d - c0, lane);
  }
}

template <typename T, int D, bool MIXED> __global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attn_dkv_kernel(Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const Place p = place(a, ROWS, 1, false);
  if (!p.on) return;
  if (MIXED && __builtin_amdgcn_readfirstlane(p.len) <= SHORT) dkv_block<T, D, MIXED>(a, p, lds);
  else dkv_block<T, D, false>(a, p, lds);
}

int64_t blocks_of(const lnx_attn_args* a, int size) { return a->nseq ? (int64_t)a->T / size + a->nseq : ((int64_t)a->T + size - 1) / size; }

// Into how many parts the rows that a block walks over are split.  In units of one tile's time in a workgroup: the launch takes as long
// as its work spread over the chip or as its longest workgroup, whichever is more; a split adds to each workgroup the time that
// its share of the result takes to be written and read in fp32 (`share`), and the joining launch.  Measured at bf16, d = 128: a tile
// 1.5 us in a workgroup with another on its CU, a share of 64 KB 5 tiles, a launch 4.  `longest`: tiles of the longest block; `most`: of
// the queries' kernels eight parts (sixteen gave nothing at any shape), of the keys', whose blocks are as long as the group's queries, sixteen
// (B1 H8/2 T1000 d128 fp32: eight 93 us, twelve 72).
int parts_for(int64_t wgs, int64_t longest, int slots, int most, double share, double launch) {
  const double work = (double)wgs * (longest + 1) / 2 / slots;
  int best = 1;
  double least = 1e300;
  for (int s = 1; s <= most && s <= longest; ++s) {
    const double extra = s > 1 ? share : 0, spread = work + extra * s * (double)wgs / slots, one = (double)((longest + s - 1) / s) + extra;
    const double t = (spread > one ? spread : one) + (s > 1 ? launch : 0);
    if (t < least * 0.95) least = t, best = s;
  }
  return best;
}
int64_t average_length(const lnx_attn_args* a) { return a->nseq ? ((int64_t)a->T + a->nseq - 1) / a->nseq : a->T; }
enum { QUERIES, DKV };  // the forward and the dq kernel, whose blocks are queries; the dk / dv kernel
int parts_of(const lnx_attn_args* a, int kernel) {
  const int64_t len = average_length(a), rows = a->nseq ? a->nseq : a->B;  // sequences of the average length
  const bool bf16 = a->dtype == LNX_BF16;
  const double share = bf16 ? 5 : 1, launch = bf16 ? 4 : 1.5;
  const int64_t keys = (len + ROWS - 1) / ROWS, queries = (len + 127) / 128;
  // workgroups that the chip holds at a time, about: two a CU, one where fp32 tiles take most of its LDS.  (The bf16 forward kernel at d > 64
  // holds three, and shares its split with the dq kernel; the model was fitted to times as it is.)
  if (kernel == DKV) return parts_for(rows * a->Hkv * keys, keys * (a->H / a->Hkv), bf16 ? 512 : 256, 16, share / 2, launch);
  return parts_for(rows * a->H * queries, keys, bf16 || a->d <= 64 ? 512 : 256, 8, share, launch);
}
// Bytes of the workspaces: shares of the forward kernel; delta and the shares of either gradient kernel
uint64_t fwd_bytes(const lnx_attn_args* a) {
  const int s = parts_of(a, QUERIES);
  return s > 1 ? (uint64_t)s * a->B * a->H * a->T * (a->d + 2) * sizeof(float) : 0;
}
uint64_t delta_bytes(const lnx_attn_args* a) { return ((uint64_t)a->B * a->H * a->T * sizeof(float) + 15) / 16 * 16; }
uint64_t bwd_bytes(const lnx_attn_args* a) {
  const int sq = parts_of(a, QUERIES), sk = parts_of(a, DKV);
  const uint64_t q = sq > 1 ? (uint64_t)sq * a->B * a->H * a->T * a->d * sizeof(float) : 0, k = sk > 1 ? (uint64_t)sk * 2 * a->B * a->Hkv * a->T * a->d * sizeof(float) : 0;
  return delta_bytes(a) + (q > k ? q : k);
}

// Rows that the kernels move as vectors, 64 of them within the 31 bits of a lane's offset.  The stride of a dimension of one element is
// never stepped over, whatever it is.
bool rows_fit(const lnx_tensor4* t, int64_t size, int B, int heads, int tokens) {
  const auto fits = [&](int extent, int64_t stride) { return extent <= 1 || stride * size % 16 == 0; };
  return (tokens <= 1 || (t->stride_t >= 0 && t->stride_t * size <= (int64_t)1 << 24)) && reinterpret_cast<uintptr_t>(t->p) % 16 == 0 && fits(B, t->stride_b) && fits(heads, t->stride_h) &&
         fits(tokens, t->stride_t);
}
int64_t stride_over(int extent, int64_t stride) { return extent > 1 ? stride : 0; }

int check(const char* what, const lnx_attn_args* a, bool bwd) {
  if (!a) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (a->B < 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->T < 0 || a->d <= 0 || a->d > 128 || a->d % 8 || a->nseq < 0 || (a->nseq && a->B != 1))
    return lnx_set_error(LNX_ERR_SHAPE, "%s: unsupported dimensions B=%d H=%d Hkv=%d T=%d d=%d nseq=%d (d a multiple of 8, at most 128; H a multiple of Hkv)", what, a->B, a->H,
                         a->Hkv, a->T, a->d, a->nseq);
  if (a->dtype != LNX_F32 && a->dtype != LNX_BF16) return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  if (a->nseq && !a->cu_seqlens) return lnx_set_error(LNX_ERR_NULL, "%s: nseq without cu_seqlens", what);
  if (a->B == 0 || a->T == 0) return LNX_OK;
  if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return lnx_set_error(LNX_ERR_SHAPE, "%s: scale must be finite", what);
  const lnx_tensor4* ts[] = {&a->q, &a->k, &a->v, &a->o, &a->d_o, &a->d_q, &a->d_k, &a->d_v};
  const int heads[] = {a->H, a->Hkv, a->Hkv, a->H, a->H, a->H, a->Hkv, a->Hkv};
  for (int i = 0; i < (bwd ? 8 : 4); ++i) {
    if (!ts[i]->p) return lnx_set_error(LNX_ERR_NULL, "%s: a tensor is missing", what);
    if (!rows_fit(ts[i], a->dtype == LNX_BF16 ? 2 : 4, a->B, heads[i], a->T)) return lnx_set_error(LNX_ERR_SHAPE, "%s: tensors must be 16-byte aligned, rows whole numbers of 16 bytes and at most 16 MiB apart", what);
  }
  if (bwd && !a->lse) return lnx_set_error(LNX_ERR_NULL, "%s: lse is required", what);
  if (a->o_low && reinterpret_cast<uintptr_t>(a->o_low) % 16) return lnx_set_error(LNX_ERR_SHAPE, "%s: o_low must be 16-byte aligned", what);
  const uint64_t need = bwd ? bwd_bytes(a) : fwd_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return lnx_set_error(LNX_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %llu bytes", what, (unsigned long long)need);
  if ((int64_t)a->B * a->H * blocks_of(a, ROWS) > MAX_GRID)  // nothing is split into parts where there are that many
    return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  return LNX_OK;
}

Args kernel_args(const lnx_attn_args* a) {
  Args k{};
  auto strides = [a](int64_t (&s)[3], const lnx_tensor4& t, int heads) {
    s[0] = stride_over(a->B, t.stride_b), s[1] = stride_over(heads, t.stride_h), s[2] = stride_over(a->T, t.stride_t);
  };
  k.q = a->q.p, k.k = a->k.p, k.v = a->v.p, k.dout = a->d_o.p, k.o = a->o.p, k.dq = a->d_q.p, k.dk = a->d_k.p, k.dv = a->d_v.p;
  strides(k.qs, a->q, a->H), strides(k.ks, a->k, a->Hkv), strides(k.vs, a->v, a->Hkv), strides(k.os, a->o, a->H);
  strides(k.gs, a->d_o, a->H), strides(k.dqs, a->d_q, a->H), strides(k.dks, a->d_k, a->Hkv), strides(k.dvs, a->d_v, a->Hkv);
  k.lse = a->lse, k.o_low = a->o_low, k.cu = a->cu_seqlens;
  k.B = a->B, k.H = a->H, k.Hkv = a->Hkv, k.G = a->H / a->Hkv, k.T = a->T, k.d = a->d, k.nseq = a->nseq, k.scale = a->scale;
  return k;
}

template <typename K> int start(K kernel, const char* name, const Args& a, int64_t grid, size_t bytes, hipStream_t st) {
  if (int rc = lnx_lds_limit(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  lnx_profile_mark(name, st);
  hipLaunchKernelGGL(kernel, dim3((unsigned)grid), dim3(256), bytes, st, a);
  return LNX_OK;
}

template <typename T, int D, bool MIXED> int launch_fwd(const lnx_attn_args* a, hipStream_t st) {
  Args k = kernel_args(a);
  k.nblk = (int)blocks_of(a, 128), k.parts = parts_of(a, QUERIES);
  const int64_t rows = (int64_t)k.B * k.H * k.T;
  k.part = static_cast<float*>(a->workspace), k.part_stat = k.part ? k.part + k.parts * rows * k.d : nullptr;
  if (int rc = start(attn_fwd_kernel<T, D, MIXED>, "attn_fwd", k, (int64_t)k.B * k.H * k.nblk * k.parts, 4 * Tile<T, D, fwd_rows<T, D>()>::BYTES + 16, st)) return rc;
  if (k.parts > 1) {
    lnx_profile_mark("attn_join", st);
    attn_join_kernel<T><<<dim3((unsigned)((rows + 15) / 16)), 256, 0, st>>>(k);
  }
  return LNX_OK;
}

template <typename T> void sum_parts(const Args& k, const float* part, int64_t stride, void* out, const int64_t (&s)[3], int heads, hipStream_t st) {
  lnx_profile_mark("attn_sum", st);
  attn_sum_kernel<T><<<dim3((unsigned)(((int64_t)k.B * heads * k.T + 15) / 16)), 256, 0, st>>>(part, k.parts, stride, static_cast<T*>(out), s[0], s[1], s[2], k.B, heads, k.T, k.d);
}

template <typename T, int D, bool MIXED> int launch_bwd(const lnx_attn_args* a, hipStream_t st) {
  Args k = kernel_args(a);
  k.delta = static_cast<float*>(a->workspace);
  k.part = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + delta_bytes(a));
  k.nblk = (int)blocks_of(a, 128), k.parts = parts_of(a, QUERIES);  // first: it leaves delta
  if (int rc = start(attn_dq_kernel<T, D, MIXED>, "attn_dq", k, (int64_t)k.B * k.H * k.nblk * k.parts, 4 * Tile<T, D>::BYTES + 16, st)) return rc;
  if (k.parts > 1) sum_parts<T>(k, k.part, (int64_t)k.B * k.H * k.T, k.dq, k.dqs, k.H, st);
  k.nblk = (int)blocks_of(a, ROWS), k.parts = parts_of(a, DKV);
  if (int rc = start(attn_dkv_kernel<T, D, MIXED>, "attn_dkv", k, (int64_t)k.B * k.Hkv * k.nblk * k.parts, 4 * Tile<T, D>::BYTES + hand_over<T>(), st)) return rc;
  if (k.parts > 1) {
    const int64_t rows = (int64_t)k.B * k.Hkv * k.T;
    sum_parts<T>(k, k.part, 2 * rows, k.dk, k.dks, k.Hkv, st);
    sum_parts<T>(k, k.part + rows * k.d, 2 * rows, k.dv, k.dvs, k.Hkv, st);
  }
  return LNX_OK;
}

template <typename T, int D, bool MIXED> int launch(const lnx_attn_args* a, bool bwd, hipStream_t st) { return bwd ? launch_bwd<T, D, MIXED>(a, st) : launch_fwd<T, D, MIXED>(a, st); }

int run(const char* what, const lnx_attn_args* a, bool bwd, hipStream_t st) {
  if (int rc = check(what, a, bwd)) return rc;
  if (a->B == 0 || a->T == 0) return LNX_OK;
  int rc;
  if (a->dtype == LNX_BF16) {
    if (a->nseq || a->T <= SHORT) rc = a->d <= 64 ? launch<bf16_t, 64, true>(a, bwd, st) : launch<bf16_t, 128, true>(a, bwd, st);
    else rc = a->d <= 64 ? launch<bf16_t, 64, false>(a, bwd, st) : launch<bf16_t, 128, false>(a, bwd, st);
  } else {
    rc = a->d <= 64 ? launch<float, 64, false>(a, bwd, st) : launch<float, 128, false>(a, bwd, st);
  }
  if (rc) return rc;
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

// ---------------------------------------------------------------------------------------------------------------
// one token against a cache
// ---------------------------------------------------------------------------------------------------------------

struct StepArgs {
  const void *q, *k, *v;
  void *kc, *vc, *o;
  const int32_t* len;
  int64_t qs[2], ks[2], vs[2], kcs[3], vcs[3];  // strides of batch, head (and place) in elements; o is dense
  float* part;  // [B H][splits][D + 2]: sums relative to a maximum, the maximum, the sum of weights
  int B, H, Hkv, G, S, d, splits, ctiles;
  float scale;
};

constexpr int SROWS = 32;  // keys of a wave's tile
template <typename T> constexpr int step_waves() { return sizeof(T) == 2 ? 4 : 2; }  // two tiles of keys and values each in LDS

// The queries that share a key head are the 32 columns, every wave walks over tiles of 32 cached tokens of its own: no barrier until
// the waves' sums meet.  Bound by the bytes of the cache (the matrix products take a sixteenth of the time): the next tile is in
// flight while one is multiplied.  The new token's key and value come from the call and are written to the cache by the wave whose
// tile holds the place; what lies behind it is never read.  bf16 weights enter the product in two parts, so that a weight is off by 2^-16
// and not by 2^-8: the products wait for the cache anyway (32 full caches of 8192 places, replayed: 195 us in one part, 197.6 in two;
// caches that lie in L2, 8 of 4096 places of 64: 21.6 and 22.6).  32 sequences of 6300 places on average, 8 key heads of 128: 155-163 us for 825
// MB, 5.1-5.3 TB/s, and 5 us to join the shares.
template <typename T, int D> __global__ __launch_bounds__(64 * step_waves<T>(), 1) void attn_step_kernel(StepArgs a) {
  constexpr int W = step_waves<T>();
  typedef Tile<T, D, SROWS> TL;
  constexpr int NI = TL::BYTES / 1024;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), n = lane & 31, kg = lane >> 5;
  int w = blockIdx.x;
  const int split = w % a.splits;
  w /= a.splits;
  const int ct = w % a.ctiles;
  w /= a.ctiles;
  const int hkv = w % a.Hkv, b = w / a.Hkv, cols = min(32, a.G - 32 * ct), h = hkv * a.G + 32 * ct + n;
  const int len = a.len[b];
  const bool good = len >= 0 && len < a.S;
  const int ntile = good ? len / SROWS + 1 : 0;
  const T* kc = static_cast<const T*>(a.kc) + b * a.kcs[0] + hkv * a.kcs[1];
  const T* vc = static_cast<const T*>(a.vc) + b * a.vcs[0] + hkv * a.vcs[1];
  const T* kn = static_cast<const T*>(a.k) + b * a.ks[0] + hkv * a.ks[1];
  const T* vn = static_cast<const T*>(a.v) + b * a.vs[0] + hkv * a.vs[1];
  char* mine = lds + wave * 4 * TL::BYTES;
  const auto kt = [&](int buf) { return reinterpret_cast<T*>(mine + 2 * buf * TL::BYTES); };
  const auto vt = [&](int buf) { return reinterpret_cast<T*>(mine + (2 * buf + 1) * TL::BYTES); };
  const auto clear = [&](void* p, int bytes) {
    for (int i = lane * 16; i < bytes; i += 1024) *reinterpret_cast<floatx4*>(static_cast<char*>(p) + i) = floatx4{0.f, 0.f, 0.f, 0.f};
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  };
  if (a.d < D) clear(mine, 4 * TL::BYTES);
  const auto fetch = [&](int tile, int buf) {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the reads of the tile that lay here
    if (tile == ntile - 1) clear(vt(buf), TL::BYTES);  // rows behind the new token: no value at all
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      int r, c;
      TL::src(j, lane, r, c);
      r += tile * SROWS;
      if (c < a.d && r <= len) {
        dma16(r < len ? kc + (int64_t)r * a.kcs[2] + c : kn + c, lds_byte_addr(kt(buf)) + 1024 * j);
        dma16(r < len ? vc + (int64_t)r * a.vcs[2] + c : vn + c, lds_byte_addr(vt(buf)) + 1024 * j);
      }
    }
  };
  const int step = a.splits * W;
  int tile = split * W + wave;
  if (tile < ntile) fetch(tile, 0);
  const float c = fmaxf(fabsf(a.scale) * LOG2E, 1e-30f);
  const T* qr = static_cast<const T*>(a.q) + b * a.qs[0] + (int64_t)(n < cols ? h : hkv * a.G) * a.qs[1];
  Frag8<T> qf[D / 16];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    from_global<T>(qf[s], qr + 16 * s + 8 * kg, 16 * s + 8 * kg < a.d && n < cols);
    if (a.scale < 0.f)
#pragma unroll
      for (int e = 0; e < 8; ++e) qf[s].v[e] = -qf[s].v[e];
  }
  floatx16 acc[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
  float m = -INFINITY, l = 0.f;
  for (int buf = 0; tile < ntile; tile += step, buf ^= 1) {
    if (tile + step < ntile) fetch(tile + step, buf ^ 1);
    if (tile + step < ntile - 1) dma_wait<2 * NI>();
    else dma_wait<0>();  // the last tile may be short of rows, and of loads
    const unsigned rows = lds_byte_addr(kt(buf)) + TL::rows(lane), cols = lds_byte_addr(kt(buf)) + TL::cols(lane);
    if (tile == ntile - 1 && ct == 0) {  // the new token's place
      T* kw = const_cast<T*>(kc) + (int64_t)len * a.kcs[2];
      T* vw = const_cast<T*>(vc) + (int64_t)len * a.vcs[2];
      for (int i = lane; i < a.d; i += 64) kw[i] = kn[i], vw[i] = vn[i];
    }
    floatx16 sc;
#pragma unroll
    for (int e = 0; e < 16; ++e) sc[e] = 0.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) mma(sc, TL::by_row(rows, 0, s), qf[s]);
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      if (tile * SROWS + frag_row(e, lane) > len) sc[e] = -INFINITY;
      top = fmaxf(top, sc[e]);
    }
    top = half_max(top);
    const float next = fmaxf(m, top), ref = next == -INFINITY ? 0.f : next * c;
    const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m * c - ref);
    m = next;
    l *= f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      sc[e] = __builtin_amdgcn_exp2f(sc[e] * c - ref);
      l += sc[e];
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][e] *= f;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      Frag8<T> pf, rest;
      from_acc(pf, sc, s);
      rest_of<true>(rest, sc, s, pf);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        const Frag8<T> v = TL::by_col(cols, TL::BYTES + 16 * s * TL::ROWB, i);
        mma(acc[i], v, pf);
        if constexpr (sizeof(T) == 2) mma(acc[i], v, rest);
      }
    }
  }
  // the waves' sums, and this workgroup's share of the result
  __syncthreads();
  float* sums = reinterpret_cast<float*>(lds);            // [W][D / 32][16][64]
  float* stat = sums + W * (D / 32) * 16 * 64;            // [W][2][32]
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) sums[((wave * (D / 32) + i) * 16 + e) * 64 + lane] = acc[i][e];
  l = xor32_sum(l);
  if (kg == 0) stat[wave * 64 + n] = m, stat[wave * 64 + 32 + n] = l;
  __syncthreads();
  float top = stat[n], sum = 0.f, f[W];
#pragma unroll
  for (int i = 1; i < W; ++i) top = fmaxf(top, stat[i * 64 + n]);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float mi = stat[i * 64 + n];
    f[i] = mi == -INFINITY && top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((mi - top) * c);
    sum += stat[i * 64 + 32 + n] * f[i];
  }
  if (n >= cols) return;
  const int64_t row = (int64_t)b * a.H + h;
  if (!good) sum = NAN;  // no place for the token: no result either
  for (int i = wave; i < D / 32; i += W)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      floatx4 t;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        t[e] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) t[e] += sums[((j * (D / 32) + i) * 16 + 4 * g + e) * 64 + lane] * f[j];
      }
      const int col = 32 * i + 8 * g + 4 * kg;
      if (a.splits == 1) {
        if (col < a.d) store4(static_cast<T*>(a.o) + row * a.d + col, floatx4{t[0] / sum, t[1] / sum, t[2] / sum, t[3] / sum});
      } else {
        store4(a.part + (row * a.splits + split) * (D + 4) + col, t);
      }
    }
  if (a.splits > 1 && wave == 0 && kg == 0) {
    float* q = a.part + (row * a.splits + split) * (D + 4) + D;
    q[0] = top * c;
    q[1] = sum;
  }
}

// One workgroup per head joins its splits (1024 at most): the factors once, then every wave adds up shares of its own, eight loads in flight
constexpr int MOST_SPLITS = 1024;
template <typename T, int D> __global__ __launch_bounds__(1024) void attn_step_join_kernel(const float* part, T* o, int splits, int d) {
  constexpr int M = D / 64;
  __shared__ float factor[MOST_SPLITS], red[16][M][64];
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const float* p = part + row * splits * (D + 4);
  float top = -INFINITY, sum = 0.f, t[M];
  for (int s = lane; s < splits; s += 64) top = fmaxf(top, p[s * (D + 4) + D]);  // every wave on its own: one barrier less
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k, LNX_WAVE));
  for (int s = lane; s < splits; s += 64) {
    const float f = top == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(p[s * (D + 4) + D] - top);
    if (wave == 0) factor[s] = f;
    sum += p[s * (D + 4) + D + 1] * f;
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k, LNX_WAVE);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < M; ++i) t[i] = 0.f;
  for (int s0 = wave; s0 < splits; s0 += 8 * waves) {
    float v[8][M];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < M; ++i) v[u][i] = s0 + u * waves < splits ? p[(s0 + u * waves) * (D + 4) + 64 * i + lane] : 0.f;
#pragma unroll
    for (int u = 0; u < 8; ++u)
      if (s0 + u * waves < splits)
#pragma unroll
        for (int i = 0; i < M; ++i) t[i] += v[u][i] * factor[s0 + u * waves];
  }
  if (waves > 1) {
#pragma unroll
    for (int i = 0; i < M; ++i) red[wave][i][lane] = t[i];
    __syncthreads();
    if (wave > 0) return;
    for (int w = 1; w < waves; ++w)
#pragma unroll
      for (int i = 0; i < M; ++i) t[i] += red[w][i][lane];
  }
#pragma unroll
  for (int i = 0; i < M; ++i)
    if (64 * i + lane < d) o[row * d + 64 * i + lane] = from_f32<T>(t[i] / sum);
}

// Splits of a cache: workgroups for four to a CU, but two tiles a wave at least of a cache that is full
int step_splits(const lnx_attn_step_args* a) {
  const int waves = a->dtype == LNX_BF16 ? step_waves<bf16_t>() : step_waves<float>();
  const int64_t wgs = (int64_t)a->B * a->Hkv * ((a->H / a->Hkv + 31) / 32), tiles = ((int64_t)a->S + SROWS - 1) / SROWS;
  int64_t s = (MOST_SPLITS + wgs - 1) / wgs;
  const int64_t most = (tiles + 2 * waves - 1) / (2 * waves);
  if (s > most) s = most;
  return (int)(s < 1 ? 1 : s);
}

// Threads of the joining workgroups: a wave for four shares
int join_threads(int splits) { return 64 * (splits <= 4 ? 1 : splits >= 64 ? 16 : (splits + 3) / 4); }

int check_step(const lnx_attn_step_args* a) {
  const char* what = "attn_step";
  if (!a) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (a->B < 0 || a->H <= 0 || a->Hkv <= 0 || a->H % a->Hkv || a->S <= 0 || a->d <= 0 || a->d > 128 || a->d % 8)
    return lnx_set_error(LNX_ERR_SHAPE, "%s: unsupported dimensions B=%d H=%d Hkv=%d S=%d d=%d (d a multiple of 8, at most 128; H a multiple of Hkv)", what, a->B, a->H, a->Hkv,
                         a->S, a->d);
  if (a->dtype != LNX_F32 && a->dtype != LNX_BF16) return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  if (a->B == 0) return LNX_OK;
  if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return lnx_set_error(LNX_ERR_SHAPE, "%s: scale must be finite", what);
  const lnx_tensor4* ts[] = {&a->q, &a->k, &a->v, &a->k_cache, &a->v_cache};
  for (int i = 0; i < 5; ++i) {
    if (!ts[i]->p) return lnx_set_error(LNX_ERR_NULL, "%s: a tensor is missing", what);
    if (!rows_fit(ts[i], a->dtype == LNX_BF16 ? 2 : 4, a->B, i == 0 ? a->H : a->Hkv, i < 3 ? 1 : a->S)) return lnx_set_error(LNX_ERR_SHAPE, "%s: tensors must be 16-byte aligned, rows whole numbers of 16 bytes and at most 16 MiB apart", what);
  }
  if (!a->o || !a->lengths) return lnx_set_error(LNX_ERR_NULL, "%s: o and lengths are required", what);
  if (reinterpret_cast<uintptr_t>(a->o) % 16) return lnx_set_error(LNX_ERR_SHAPE, "%s: tensors must be 16-byte aligned, rows whole numbers of 16 bytes and at most 16 MiB apart", what);
  if ((int64_t)a->B * a->H > MAX_GRID || (int64_t)a->B * a->Hkv * ((a->H / a->Hkv + 31) / 32) * step_splits(a) > MAX_GRID) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  const uint64_t need = lnx_attn_step_workspace_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need || reinterpret_cast<uintptr_t>(a->workspace) % 16))
    return lnx_set_error(LNX_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %llu bytes", what, (unsigned long long)need);
  return LNX_OK;
}

template <typename T, int D> int launch_step(const lnx_attn_step_args* a, hipStream_t st) {
  constexpr int W = step_waves<T>();
  StepArgs k{};
  k.q = a->q.p, k.k = a->k.p, k.v = a->v.p, k.kc = a->k_cache.p, k.vc = a->v_cache.p, k.o = a->o, k.len = a->lengths, k.part = static_cast<float*>(a->workspace);
  auto strides = [a](int64_t* s, const lnx_tensor4& t, int heads) { s[0] = stride_over(a->B, t.stride_b), s[1] = stride_over(heads, t.stride_h); };
  strides(k.qs, a->q, a->H), strides(k.ks, a->k, a->Hkv), strides(k.vs, a->v, a->Hkv), strides(k.kcs, a->k_cache, a->Hkv), strides(k.vcs, a->v_cache, a->Hkv);
  k.kcs[2] = stride_over(a->S, a->k_cache.stride_t), k.vcs[2] = stride_over(a->S, a->v_cache.stride_t);
  k.B = a->B, k.H = a->H, k.Hkv = a->Hkv, k.G = a->H / a->Hkv, k.S = a->S, k.d = a->d, k.scale = a->scale;
  k.splits = step_splits(a), k.ctiles = (k.G + 31) / 32;
  const size_t tiles = W * 4 * Tile<T, D, SROWS>::BYTES, sums = W * ((D / 32) * 16 * 64 + 64) * sizeof(float), bytes = tiles > sums ? tiles : sums;
  const auto kernel = attn_step_kernel<T, D>;
  if (int rc = lnx_lds_limit(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  lnx_profile_mark("attn_step", st);
  hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)k.B * k.Hkv * k.ctiles * k.splits)), dim3(64 * W), bytes, st, k);
  if (k.splits > 1) {
    lnx_profile_mark("attn_step_join", st);
    attn_step_join_kernel<T, D><<<dim3((unsigned)((int64_t)k.B * k.H)), join_threads(k.splits), 0, st>>>(k.part, static_cast<T*>(a->o), k.splits, k.d);
  }
  return LNX_OK;
}

}  // namespace

extern "C" uint64_t lnx_attn_step_workspace_bytes(const lnx_attn_step_args* a) {
  if (!a || a->B <= 0 || a->H <= 0 || a->Hkv <= 0 || a->S <= 0) return 0;
  const int s = step_splits(a);
  return s > 1 ? (uint64_t)a->B * a->H * s * ((a->d <= 64 ? 64 : 128) + 4) * sizeof(float) : 0;
}
extern "C" int lnx_attn_step(const lnx_attn_step_args* a, void* hip_stream) {
  if (int rc = check_step(a)) return rc;
  if (a->B == 0) return LNX_OK;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  int rc;
  if (a->dtype == LNX_BF16) rc = a->d <= 64 ? launch_step<bf16_t, 64>(a, st) : launch_step<bf16_t, 128>(a, st);
  else rc = a->d <= 64 ? launch_step<float, 64>(a, st) : launch_step<float, 128>(a, st);
  if (rc) return rc;
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "attn_step: %s", hipGetErrorString(e));
}

static bool attn_sizes(const lnx_attn_args* a) { return a && a->B > 0 && a->H > 0 && a->Hkv > 0 && a->T > 0 && a->d > 0 && a->nseq >= 0; }
extern "C" uint64_t lnx_attn_fwd_workspace_bytes(const lnx_attn_args* a) { return attn_sizes(a) ? fwd_bytes(a) : 0; }
extern "C" uint64_t lnx_attn_bwd_workspace_bytes(const lnx_attn_args* a) { return attn_sizes(a) ? bwd_bytes(a) : 0; }
extern "C" int lnx_attn_fwd(const lnx_attn_args* a, void* hip_stream) { return run("attn_fwd", a, false, static_cast<hipStream_t>(hip_stream)); }
extern "C" int lnx_attn_bwd(const lnx_attn_args* a, void* hip_stream) { return run("attn_bwd", a, true, static_cast<hipStream_t>(hip_stream)); }
