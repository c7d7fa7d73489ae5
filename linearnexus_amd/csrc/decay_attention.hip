// Linear attention with a decay for each head, forward, backward and one token:
//   S_t = e^{g_t} S_{t-1} + k_t^T v_t     o_t = scale q_t S_t
//   dS_t = scale q_t^T do_t + e^{g_{t+1}} dS_{t+1}     dq_t = scale do_t S_t^T     dk_t = v_t dS_t^T     dv_t = k_t dS_t     dg_t = e^{g_t} <dS_t, S_{t-1}>
// All four results are one walk over chunks of C tokens, forwards or backwards (G: sums of g within the chunk):
//   out_i = sum_{j <= i} (x_i . y_j) e^{G_i - G_j} z_j + e^{G_i} x_i S       S <- e^{G_C} S + sum_j e^{G_C - G_j} y_j^T z_j
// with (x, y, z) = (q, k, v) for o, (do, v, k) for dq and, mirrored in time, (v, do, q) for dk and (k, q, do) for dv.  A workgroup walks 64
// columns of z: each of its four waves keeps 16 columns of the state in registers, in the layout of a product's result, which is the layout
// of the next product's operand (tile pairs of 16 x 16), so the state never leaves them.  A chunk's pairs are formed once per workgroup
// and handed over through LDS.
// Rounding (bf16): pairs, the state as an operand and the z_j with their factors enter the products in two bf16 parts or three, so results are off
// by their own rounding alone, states like fp32's, and dg, a running difference of x . out and y . out over a whole sequence, keeps its digits.
// Exponents are differences of sums over a chunk: the sums are held as a multiple of 1/64 and a rest, so that a difference is exact to a unit
// however far the sums have run (a decay of e^-100 beside one of 1).
// Measured at d128 in bf16: B8 H16 T4096 forward 141 - 165 us (537 MB, 3.3 - 3.8 TB/s), backward 577 - 640 (its three walks read 1.41 GB and write
// 0.41) and 22 for dg; one prompt of H16 T65000 147 + 8 + 306; a token at B256 H32 210 us, 5.1 TB/s.  A walk's bound is what its eight waves issue:
// of a chunk's 5400 cycles (7200 where dg is taken) vector instructions hold a SIMD for 49 %, the matrix cores for 30 (26), and a CU, whose LDS one
// workgroup fills, has two waves a SIMD to put between each other.

#include <type_traits>

#include "lnx_common.h"
#include "lds_direct.h"
#include "mma_tiles.h"
#include "packed_slots.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SLAB = 64;                        // columns of z of a workgroup: 16 a wave
constexpr int64_t MAX_GRID = 0xffffffff;        // threads of a launch
constexpr int WALK_THREADS = 512, JOIN_THREADS = 256, GATE_THREADS = 1024, STEP_THREADS = 256;
typedef __attribute__((address_space(3))) char lds_char;

// Products of 16 x 16 tiles: K contraction slots an operand, which the results of TP tiles fill.  Slot (a, r) of lane group g = lane / 16 is
// index 16 a + 4 g + r of the K: element r of that group in result tile a.
template <typename T> struct Form;
template <> struct Form<bf16_t> {
  static constexpr int K = 32, TP = 2;
  typedef bf16x8 Frag;
  static __device__ __forceinline__ void mma(floatx4& c, const Frag& a, const Frag& b) { c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ void put(Frag& f, int a, int r, float x) { f[4 * a + r] = (bf16_t)x; }
  static __device__ __forceinline__ float get(const Frag& f, int a, int r) { return (float)f[4 * a + r]; }
};
template <> struct Form<float> {
  static constexpr int K = 16, TP = 1;
  typedef floatx4 Frag;
  static __device__ __forceinline__ void mma(floatx4& c, const Frag& a, const Frag& b) {
#pragma unroll
    for (int r = 0; r < 4; ++r) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], b[r], c, 0, 0, 0);
  }
  static __device__ __forceinline__ void put(Frag& f, int, int r, float x) { f[r] = x; }
  static __device__ __forceinline__ float get(const Frag& f, int, int r) { return f[r]; }
};
// Tokens of a chunk: three of them lie in LDS at a time
template <typename T, int KW> constexpr int chunk_of() { return (sizeof(T) == 2 ? 64 : 32) / (KW > 128 ? 2 : 1); }
__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Result tiles as an operand in P parts: each is rounded to bf16 and the next holds what that left.  Of an infinite value that is not a number: as
// an integer it lies above 2^100, where rests are cut (two at a time), so that it adds nothing to a sum that the infinite value is in.
__device__ __forceinline__ floatx4 minus(floatx4 v, bf16x4 h) { return floatx4{v[0] - (float)h[0], v[1] - (float)h[1], v[2] - (float)h[2], v[3] - (float)h[3]}; }
__device__ __forceinline__ bf16x4 rest(floatx4 d) {
  typedef short short4_ __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(bf16x4, __builtin_elementwise_min(__builtin_bit_cast(short4_, pack_bf16x4(d)), short4_{0x7180, 0x7180, 0x7180, 0x7180}));
}
// Rounded to bf16, and opaque: -ffast-math takes a conversion and its inverse for nothing, and the rest with them
__device__ __forceinline__ bf16x4 to_bf16(floatx4 v) {
  typedef unsigned uint2_ __attribute__((ext_vector_type(2)));
  uint2_ u = __builtin_bit_cast(uint2_, pack_bf16x4(v));
  asm("" : "+v"(u));
  return __builtin_bit_cast(bf16x4, u);
}
template <int P> __device__ __forceinline__ void parts_of(floatx4 v, bf16x4 (&part)[P]) {
  part[0] = to_bf16(v);
#pragma unroll
  for (int i = 1; i < P; ++i) {
    v = minus(v, part[i - 1]);
    part[i] = rest(v);
  }
}
template <int P> __device__ __forceinline__ void split(const floatx4 (&v)[2], bf16x8 (&part)[P]) {
  bf16x4 a[P], b[P];
  parts_of(v[0], a);
  parts_of(v[1], b);
#pragma unroll
  for (int i = 0; i < P; ++i) part[i] = Mma16::join(a[i], b[i]);
}
__device__ __forceinline__ void split(const floatx4 (&v)[1], floatx4 (&part)[1]) { part[0] = v[0]; }

// Whether all of an operand's values are finite: their exponents, two of bf16 at a time
__device__ __forceinline__ bool all_finite(const bf16x8& f) {
  typedef unsigned uint4_ __attribute__((ext_vector_type(4)));
  const uint4_ u = __builtin_bit_cast(uint4_, f);
  unsigned any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) any |= (u[i] & 0x7f807f80u) + 0x00800080u;
  return !(any & 0x80008000u);
}
__device__ __forceinline__ bool all_finite(const floatx4& f) { return is_finite(f[0]) && is_finite(f[1]) && is_finite(f[2]) && is_finite(f[3]); }

// A [C][W] tile in LDS as loads that go straight there leave it: 16-byte granules of a row permuted by an exclusive or with x(row), chosen so that
// row operands (16 consecutive rows, one granule) and column operands (the transposing reads of two lane groups: 8 consecutive rows, 2 granules;
// fp32: rows 4 g + r for one r, 4 granules) touch every bank once.  x depends on row % 16 only.
template <typename V> __device__ __forceinline__ V lds_load(unsigned addr) { return *(__attribute__((address_space(3))) const V*)(lds_char*)(uintptr_t)addr; }
template <typename T, int W> struct Cells;
template <int W> struct Cells<bf16_t, W> {
  static constexpr int ROWB = 2 * W, G = W / 8;
  static __device__ __forceinline__ int x(int r) { return G == 8 ? (r & 6) | ((r >> 3) & 1) : ((r & 3) << 2) | ((r >> 1) & 2) | ((r >> 3) & 1); }
  static __device__ __forceinline__ void src(int p, int& r, int& c) {  // row and first column of granule p of the tile's memory
    r = p / G;
    c = ((p % G) ^ x(r)) << 3;
  }
  static __device__ __forceinline__ unsigned rows(int lane) {
    const int r = lane & 15, g = lane >> 4;
    return r * ROWB + (((g >> 1) ^ x(r)) << 4) + 8 * (g & 1);
  }
  // columns K s + slots of the row that `rows` points at; `off`: whole groups of 16 rows, tiles
  static __device__ __forceinline__ bf16x8 by_row(unsigned rows, int off, int s) {
    typedef float float2_ __attribute__((ext_vector_type(2)));
    typedef const volatile __attribute__((address_space(3))) float2_ lds_float2;  // (kept apart: one ds_read2_b64 takes longer than two ds_read_b64)
    const float2_ lo = *(lds_float2*)(lds_char*)(uintptr_t)((rows ^ (64 * s)) + off), hi = *(lds_float2*)(lds_char*)(uintptr_t)((rows ^ (64 * s + 32)) + off);
    return Mma16::join(__builtin_bit_cast(bf16x4, lo), __builtin_bit_cast(bf16x4, hi));
  }
  static __device__ __forceinline__ unsigned cols(int lane) {
    const int s = lane & 15, r = 4 * (lane >> 4) + (s >> 2);
    return r * ROWB + ((((s >> 1) & 1) ^ x(r)) << 4) + 8 * (s & 1);
  }
  // rows k0 + slots of column 16 i + (lane & 15)
  static __device__ __forceinline__ bf16x8 by_col(unsigned cols, int k0, int i) {
    typedef short short4_ __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4_ lds_short4;
    const unsigned at = (cols ^ (32 * i)) + k0 * ROWB;
    return Mma16::join(__builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds_char*)(uintptr_t)at)),
                       __builtin_bit_cast(bf16x4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(lds_char*)(uintptr_t)(at + 16 * ROWB))));
  }
};
template <int W> struct Cells<float, W> {
  static constexpr int ROWB = 4 * W, G = W / 4;
  static __device__ __forceinline__ int x(int r) { return (r & 12) | (r & 3); }
  static __device__ __forceinline__ void src(int p, int& r, int& c) {
    r = p / G;
    c = ((p % G) ^ x(r)) << 2;
  }
  static __device__ __forceinline__ unsigned rows(int lane) {
    const int r = lane & 15;
    return r * ROWB + (((lane >> 4) ^ x(r)) << 4);
  }
  static __device__ __forceinline__ floatx4 by_row(unsigned rows, int off, int s) { return lds_load<floatx4>((rows ^ (64 * s)) + off); }
  static __device__ __forceinline__ unsigned cols(int lane) {
    const int l = lane & 15, g = lane >> 4;
    return 4 * g * ROWB + (((l >> 2) ^ (4 * g)) << 4) + 4 * (l & 3);
  }
  static __device__ __forceinline__ floatx4 by_col(unsigned cols, int k0, int i) {
    floatx4 f;
#pragma unroll
    for (int r = 0; r < 4; ++r) f[r] = lds_load<float>((cols ^ (16 * r) ^ (64 * i)) + (k0 + r) * ROWB);
    return f;
  }
};

// Of two values the sums over pairs of rows of 16 lanes (over the halves): even rows (the lower half) get the first's, odd ones the second's
__device__ __forceinline__ float rows_join16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float rows_join32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Sum over the lanes up to this one
template <int CTRL, int ROWS> __device__ __forceinline__ float from_lane(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ float running_sum(float x) {
  x += from_lane<0x111, 0xF>(x);  // row_shr:1, 2, 4, 8
  x += from_lane<0x112, 0xF>(x);
  x += from_lane<0x114, 0xF>(x);
  x += from_lane<0x118, 0xF>(x);
  x += from_lane<0x142, 0xA>(x);  // row_bcast:15 into rows 1 and 3
  x += from_lane<0x143, 0xC>(x);  // row_bcast:31 into rows 2 and 3
  return x;
}
__device__ __forceinline__ float lane_value(float x, int lane) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), lane)); }

// A value as it is, which the compiler may not regroup or fuse with what takes it
__device__ __forceinline__ float rounded(float x) {
  asm("" : "+v"(x));
  return x;
}
// 2^(difference of two sums), each a multiple of 1/64 and a rest
__device__ __forceinline__ float between(float h1, float l1, float h0, float l0) { return __builtin_amdgcn_exp2f(rounded(h1 - h0) + (l1 - l0)); }

struct Side {
  void* p;
  int64_t sb, sh, st;  // strides of batch, head and token in elements
};
// One walk.  The state is [width of y][width of z]; in memory always [dk][dv], `turned` says that y runs along dv.
struct Role {
  Side x, y, z, w, out;  // w: what the results are multiplied with for dg
  int kw, vw;            // widths of x and y, of z and out
  int sk, sn;            // the state's, which the tensors may exceed by columns of zeros
  int rev, turned, slabs;
  float row_scale, col_scale;  // of a state's part of the results; of what a token adds to the state
  const float* init;
  float* fin;
  float* dots;  // [inter, pairs][slab][B H][T]
};
struct Walk {
  Role role[3];
  const float* g;
  int64_t gb, gh, gt;
  const int32_t* cu;
  float* whole;      // local walks: every segment's factor e^{sum g}, [slot][H]
  int B, H, T, nseq, dv;
  int seg, nseg;     // tokens of a segment; segments of a dense row
  int by_slot;       // init is per segment, not per row
  int units, per;    // (slot, head) pairs; workgroups of each
  int64_t dots_step; // from one slab's dots to the next
  float scale;
};

// Where a segment lies: its row (batch row or sequence), first token, length; whether it is its row's first or last
struct Spot {
  int b, row, len;
  int64_t tok;
  bool on, first, last;
};
template <typename A> __device__ __forceinline__ Spot spot(const A& a, int slot) {
  Spot s;
  if (!a.nseq) {
    s.b = s.row = slot / a.nseg;
    const int i = slot % a.nseg;
    s.tok = (int64_t)i * a.seg;
    s.len = min(a.seg, a.T - (int)s.tok);
    s.on = true, s.first = i == 0, s.last = i == a.nseg - 1;
    return s;
  }
  s.b = 0;
  s.row = packed_owner(a.cu, a.nseq, a.T, a.seg, slot);
  const int from = seq_first(a.cu, s.row, a.T), len = seq_end(a.cu, s.row, a.T) - from;
  const int n = max(1, (int)(((unsigned)len + a.seg - 1) / a.seg)), i = (int)(slot - packed_slot(from, s.row, a.seg));
  s.tok = from + (int64_t)i * a.seg;
  s.len = min(a.seg, len - i * a.seg);
  s.on = i >= 0 && i < n, s.first = i == 0, s.last = i == n - 1;
  return s;
}

// Brings [C][W] tiles to LDS by four waves; which bytes a lane fetches is formed once.
template <typename T, int W, int C> struct Mover {
  typedef Cells<T, W> CL;
  static constexpr int N = C * CL::ROWB / 1024 / 4;
  unsigned off[N];
  __device__ __forceinline__ Mover(int64_t st, int wave, int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      int r, c;
      CL::src(64 * (wave * N + i) + lane, r, c);
      off[i] = (unsigned)((r * (int)st + c) * (int)sizeof(T));
    }
  }
  // Rows from `base` on, all of them there: load i of this wave's
  __device__ __forceinline__ void one(int i, unsigned tile, const T* base, int wave) const { dma16_at(base, off[i], tile + 1024 * (wave * N + i)); }
  // Rows behind the last of `valid` are copies of it, columns behind `width` keep the zeros that lie there
  __device__ __forceinline__ void edge(unsigned tile, const T* base, int64_t st, int valid, int width, int wave, int lane) const {
#pragma unroll 1
    for (int i = 0; i < N; ++i) {
      int r, c;
      CL::src(64 * (wave * N + i) + lane, r, c);
      if (c < width) dma16(base + (int64_t)min(r, valid - 1) * st + c, tile + 1024 * (wave * N + i));
    }
  }
};

template <typename T> __device__ __forceinline__ const T* head_of(const Side& s, const Spot& p, int h) {
  return static_cast<const T*>(s.p) + p.b * s.sb + h * s.sh + p.tok * s.st;
}

// bf16 parts of an operand that is not one of the inputs.  What a token adds to the state: three, exact as fp32 is.  The state as an operand and the
// pairs: three where dg is taken from the results, two where they are rounded to bf16.  (Errors against 64 bits, all in two parts -> thus: states
// of H8 T4096 d128 2.4e-6 -> 2.2e-7, dg 1.4e-6 -> 2.2e-7 by the state's; dg per head of B10 H3 T40 6.3e-6 -> 2.9e-7 by the pairs'.  B8 H16 T4096, us:
// forward 151 -> 165, backward 530 -> 650, 575 without the state's third part, 620 without the pairs'.)
template <typename T> constexpr int parts_of_z() { return sizeof(T) == 2 ? 3 : 1; }
template <typename T> constexpr int parts_of_state(bool dots) { return sizeof(T) == 2 ? (dots ? 3 : 2) : 1; }
template <typename T> constexpr int parts_of_pairs(bool dots) { return sizeof(T) == 2 ? (dots ? 3 : 2) : 1; }

// LDS of a walk.  OUT: false for the local walks of segments, which leave what a segment adds to the state and nothing else.  BWD: walks with dots among them.
template <typename T, int KW, bool OUT, bool BWD> struct Room {
  static constexpr int C = chunk_of<T, KW>(), NI = C / 16, NJ = C / Form<T>::K;
  // Pairs lie in LDS as operands, in blocks of 16 rows x K: those that have any, of bf16 in half a block where only one of its two tiles has
  static constexpr bool needed(int i, int j, bool rev) { return rev ? Form<T>::K * (j + 1) > 16 * i : Form<T>::K * j <= 16 * i + 15; }
  static constexpr bool half(int i, int j, bool rev) { return Form<T>::TP == 2 && (rev ? 2 * j < i : 2 * j + 1 > i); }
  static constexpr int P = parts_of_pairs<T>(BWD);
  static constexpr int block(int i, int j, bool rev) {  // where block (i, j) begins
    int at = 0;
    for (int b = 0; b < i * NJ + j; ++b)
      if (needed(b / NJ, b % NJ, rev)) at += P * (half(b / NJ, b % NJ, rev) ? 512 : 1024);
    return at;
  }
  static constexpr int slot(int i, int j, bool rev) {  // its number
    int n = 0;
    for (int b = 0; b < i * NJ + j; ++b) n += needed(b / NJ, b % NJ, rev);
    return n;
  }
  static constexpr int SLOTS = slot(NI, 0, false);
  static constexpr int XB = C * KW * sizeof(T), ZB = C * SLAB * sizeof(T), BUF = (OUT ? 2 : 1) * XB + ZB, PAIRB = OUT ? block(NI, 0, false) : 0;
  static constexpr int RING = OUT ? 3 : 6, AHEAD = RING - 1;  // chunks in LDS; how far ahead they are fetched (their gates one more)
  static constexpr int PAIRS = RING * BUF, FACTORS = PAIRS + PAIRB, SUMS = FACTORS + 2 * 1024, RAW = SUMS + 4 * 512, DOTS = RAW + (RING + 1) * 256;
  static constexpr int BYTES = DOTS + (OUT ? 2 * 4 * 2 * C * 4 : 0);
  // The 16 x 16 tiles of pairs, ten of a chunk of 64, in four nearly equal shares: tile u of wave w
  static constexpr int units(int w) { return NI == 4 ? (w < 2 ? 2 : 3) : w < NI * (NI + 1) / 2; }
  static constexpr int unit_row(int w, int u, bool rev) {
    const int i = NI == 4 ? (w == 0 ? 3 * u : w) : w > 0;
    return rev ? NI - 1 - i : i;
  }
  static constexpr int unit_col(int w, int u, bool rev) {
    const int j = NI == 4 ? (w == 0 ? 0 : w == 3 ? u + 1 : u) : w == 2;
    return rev ? NI - 1 - j : j;
  }
};

// What a workgroup works on
struct Task {
  Spot p;
  int slot, h, item, nchunk, col0, vw;  // vw: columns of its slab that exist
};
template <bool REV> __device__ __forceinline__ int chunk_at(const Task& k, int it) { return REV ? k.nchunk - 1 - it : it; }

// Scheduling of a stretch of MFMAS matrix instructions: VALUS vector instructions behind each of them.  Left to itself the compiler puts what can run
// beside a matrix instruction (16 cycles) before or behind the whole run.
template <typename T, int MFMAS, int VALUS> __device__ __forceinline__ void interleave() {
  if constexpr (sizeof(T) == 2) {
#pragma unroll
    for (int i = 0; i < MFMAS; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x2, VALUS, 0);
    }
  }
}

// Four of a walk's eight waves.  While the others take what the state gives, they form the chunk's pairs, a share of the tiles each; while the others
// take what the pairs give and move the state on, they send for the chunk after next and form the next one's decays.  Two barriers a chunk.  (With one, the
// pairs a chunk ahead of the state and the loads one chunk ahead of them: B8 H16 T4096 d128 forward 162 us -> 159, backward 644 -> 638.)
template <typename T, int KW, bool OUT, bool REV, bool BWD, int W> __device__ __forceinline__ void walk_pairs(const Walk& a, const Role& ro, const Task& k, char* lds) {
  typedef Form<T> F;
  typedef typename F::Frag Frag;
  typedef Cells<T, KW> XC;
  typedef Room<T, KW, OUT, BWD> R;
  constexpr int C = R::C, NS = KW / F::K;
  constexpr int wave = W, UNITS = R::units(W);
  const int lane = threadIdx.x & 63, l16 = lane & 15, g4 = 4 * (lane >> 4);
  const Spot& p = k.p;
  const unsigned lds0 = lds_byte_addr(lds);
  // Where the next chunk lies: what a lane fetches is at a fixed offset from these
  const int64_t dir = REV ? -C : C;
  const int first = chunk_at<REV>(k, 0) * C;
  const T* xp = OUT ? head_of<T>(ro.x, p, k.h) + first * ro.x.st : nullptr;
  const T* yp = head_of<T>(ro.y, p, k.h) + first * ro.y.st;
  const T* zp = head_of<T>(ro.z, p, k.h) + k.col0 + first * ro.z.st;
  const int64_t x_step = OUT ? dir * ro.x.st : 0, y_step = dir * ro.y.st, z_step = dir * ro.z.st, g_step = dir * a.gt;
  const float* gp = a.g + p.b * a.gb + k.h * a.gh + (p.tok + first + min(lane, C - 1)) * a.gt;
  int g_next = first, raw_next = 0;  // the next chunk of gates: its first token, its place
  const Mover<T, KW, C> mx(OUT ? ro.x.st : 0, wave, lane), my(ro.y.st, wave, lane);
  const Mover<T, SLAB, C> mz(ro.z.st, wave, lane);
  const bool wide = ro.kw >= KW && k.vw == SLAB;
  int t_next = first;  // the next chunk's first token
  // A chunk's loads, ten of a wave at KW = 128, all at once: a CU takes 64 bytes a cycle, for which these waves wait (of 40 KB 640 cycles), but
  // handed out between the steps of their work they kept the last ones from the next chunk (forward at B8 H16 T4096 d128, one chunk ahead, 157 us -> 178 - 210)
  constexpr int NX = OUT ? decltype(mx)::N : 0, NY = decltype(my)::N, NZ = decltype(mz)::N;
  const auto fetch = [&](int buf) {
    const int valid = min(C, p.len - t_next);
    const unsigned tiles = lds0 + buf * R::BUF;
    if (valid == C && wide) {
#pragma unroll
      for (int i = 0; i < NY + NX + NZ; ++i) {
        if (i < NY) my.one(i, tiles, yp, wave);
        else if (i < NY + NX) mx.one(OUT ? i - NY : 0, tiles + R::XB + R::ZB, xp, wave);
        else mz.one(i - NY - NX, tiles + R::XB, zp, wave);
      }
    } else {
      my.edge(tiles, yp, ro.y.st, valid, ro.kw, wave, lane);
      if constexpr (OUT) mx.edge(tiles + R::XB + R::ZB, xp, ro.x.st, valid, ro.kw, wave, lane);
      mz.edge(tiles + R::XB, zp, ro.z.st, valid, k.vw, wave, lane);
    }
    yp += y_step, xp += x_step, zp += z_step, t_next += (int)dir;
  };
  const auto fetch_gates = [&] {
    if (wave == 0) dma4(gp - max(0, min(lane, C - 1) - (min(C, p.len - g_next) - 1)) * a.gt, lds0 + R::RAW + 256 * raw_next);
    gp += g_step, g_next += (int)dir, raw_next = raw_next == R::RING ? 0 : raw_next + 1;
  };
  // the dots of the chunk before the one that is walked: thread = (kind, token)
  const float* red = reinterpret_cast<const float*>(lds + R::DOTS);
  const bool dots = OUT && ro.dots;
  const int dot_i = (threadIdx.x - 256) % C, dot_kind = (threadIdx.x - 256) / C;
  int dot_t = first + dot_i;
  float* dot_p = dots && dot_kind < 2 ? ro.dots + (int64_t)(dot_kind * ro.slabs + k.item) * a.dots_step + (int64_t)(p.b * a.H + k.h) * a.T + p.tok + dot_t : nullptr;
  const auto leave_dots = [&](int it) {
    if (dot_p && dot_t < p.len) {
      const float* q = red + (it & 1) * 8 * C + dot_kind * C + dot_i;
      *dot_p = (q[0] + q[2 * C]) + (q[4 * C] + q[6 * C]);
    }
    dot_p += dot_p ? dir : 0;
    dot_t += (int)dir;
  };
  float* sums = reinterpret_cast<float*>(lds + R::SUMS) + 128 * wave;  // of this wave: multiples, rests
  const float* raw = reinterpret_cast<const float*>(lds + R::RAW);
  float whole_h = 0.f, whole_l = 0.f;
  // until chunk `it` is there: all but the loads of those behind it.  Their number is the same whatever the widths: a load covers whole rows, whose first
  // granules lie within any width, so that none of a tile's loads is without lanes.  (Waiting for all of them where a width fills no tile: B8 H16 T4096 dk 80, dv 96 in
  // bf16 forward 196 us -> 220, backward 731 -> 796.)
  const auto arrived = [&](int it) {
    constexpr int N = (R::AHEAD - 1) * (NY + NX + NZ);
    if (it + R::AHEAD < k.nchunk) dma_wait<wave == 0 ? N + R::AHEAD - 1 : N>();
    else dma_wait<0>();
  };
  const auto decays = [&](int it, int raw_at, int t0) {  // lane = token
    const int valid = min(C, p.len - t0);
    float gv = lane < valid ? raw[64 * raw_at + lane] * LOG2E : 0.f;
    gv = gv < -200.f ? -200.f : gv;  // e^-138 is nothing
    const float gm = rounded(rintf(gv * 64.f) * (1.f / 64.f)), H = running_sum(gm), L = running_sum(gv - gm), HT = lane_value(H, 63), LT = lane_value(L, 63);
    sums[lane] = H;
    sums[64 + lane] = L;
    if (wave == 3) {
      const float head = between(H, L, 0.f, 0.f), tail = between(HT, LT, H, L);
      float* f = reinterpret_cast<float*>(lds + R::FACTORS) + 256 * (it & 1);
      f[lane] = (REV ? tail : head) * ro.row_scale;
      f[64 + lane] = lane < valid ? (REV ? head : tail) * ro.col_scale : 0.f;
      f[128 + lane] = between(HT, LT, 0.f, 0.f);
      if (!OUT) whole_h += HT, whole_l += LT;
    }
  };
  for (int i = 0; i <= R::AHEAD && i < k.nchunk; ++i) fetch_gates();
  for (int i = 0; i < R::AHEAD && i < k.nchunk; ++i) fetch(i);
  dma_wait<0>();
  lds_barrier();
  if (k.nchunk > 0) decays(0, 0, first);
  lds_barrier();
  for (int it = 0, buf = 0, raw_at = 0, t0 = first; it < k.nchunk; ++it) {
    if (dots && it >= 1) leave_dots(it - 1);  // (ahead of the loads, so that those still on their way at the wait below are loads alone: it is waited for there)
    if constexpr (OUT) {
      if constexpr (UNITS > 0) {
        // ---- pairs: rows of a result are j, its column is i
        constexpr bool TWO_ROWS = UNITS > 1 && R::unit_row(W, 0, REV) != R::unit_row(W, UNITS > 1, REV);  // (wave 0's)
        Frag x[1 + TWO_ROWS][NS], y[UNITS][NS];
        const unsigned xr = lds0 + buf * R::BUF + R::XB + R::ZB + XC::rows(lane), yr = lds0 + buf * R::BUF + XC::rows(lane);
#pragma unroll
        for (int s = 0; s < NS; ++s) {
#pragma unroll
          for (int u = 0; u < UNITS; ++u) {
            if (u <= TWO_ROWS) x[u][s] = XC::by_row(xr, R::unit_row(W, u, REV) * 16 * XC::ROWB, s);
            y[u][s] = XC::by_row(yr, R::unit_col(W, u, REV) * 16 * XC::ROWB, s);
          }
        }
        const int valid = min(C, p.len - t0);
        char* pairs = lds + R::PAIRS;
        floatx4 sc[UNITS], w[UNITS];
        // what the decays make of them is formed beside the reads
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const int i = 16 * R::unit_row(W, u, REV) + l16, j0 = 16 * R::unit_col(W, u, REV) + g4;
          const float hi_ = sums[i], li_ = sums[64 + i];
          const floatx4 hj = load4(sums + j0), lj = load4(sums + 64 + j0);
#pragma unroll
          for (int r = 0; r < 4; ++r) w[u][r] = REV ? between(hj[r], lj[r], hi_, li_) : between(hi_, li_, hj[r], lj[r]);
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u) sc[u] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
          for (int u = 0; u < UNITS; ++u) F::mma(sc[u], y[u][s], x[u < 1 + TWO_ROWS ? u : TWO_ROWS][s]);
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const int it16 = R::unit_row(W, u, REV), jt = R::unit_col(W, u, REV), i = 16 * it16 + l16, j0 = 16 * jt + g4;
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[u][r] *= w[u][r];
          if (it16 == jt || (REV && valid < C)) {
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[u][r] = (REV ? j0 + r >= i && j0 + r < valid : j0 + r <= i) ? sc[u][r] : 0.f;
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[u][r] = rounded(sc[u][r]);
          const bool half = R::half(it16, jt / F::TP, REV);
          char* q = pairs + R::block(it16, jt / F::TP, REV) + (half ? 8 : 16) * lane;
          if constexpr (F::TP == 2) {
            bf16x4 part[R::P];
            parts_of(sc[u], part);
#pragma unroll
            for (int i = 0; i < R::P; ++i) *reinterpret_cast<bf16x4*>(q + (half ? 512 * i : 8 * (jt % 2) + 1024 * i)) = part[i];
          } else {
            *reinterpret_cast<floatx4*>(q) = sc[u];
          }
        }
      }
      lds_barrier();
    }
    if (it + R::AHEAD < k.nchunk) fetch(buf == 0 ? R::RING - 1 : buf - 1);
    if (it + R::AHEAD + 1 < k.nchunk) fetch_gates();
    buf = buf == R::RING - 1 ? 0 : buf + 1;
    raw_at = raw_at == R::RING ? 0 : raw_at + 1;
    t0 += (int)dir;
    if (it + 1 < k.nchunk) decays(it + 1, raw_at, t0);
    arrived(it + 1);
    lds_barrier();
  }
  if (dots && k.nchunk > 0) leave_dots(k.nchunk - 1);
  if (!OUT && k.item == 0 && threadIdx.x == 448) a.whole[(int64_t)k.slot * a.H + k.h] = between(whole_h, whole_l, 0.f, 0.f);
}

template <typename T, int KW, bool OUT, bool REV, bool BWD> __device__ __forceinline__ void pair_wave(int wave, const Walk& a, const Role& ro, const Task& k, char* lds) {
  if (wave == 0) walk_pairs<T, KW, OUT, REV, BWD, 0>(a, ro, k, lds);
  else if (wave == 1) walk_pairs<T, KW, OUT, REV, BWD, 1>(a, ro, k, lds);
  else if (wave == 2) walk_pairs<T, KW, OUT, REV, BWD, 2>(a, ro, k, lds);
  else walk_pairs<T, KW, OUT, REV, BWD, 3>(a, ro, k, lds);
}

// The other four: 16 columns of the state and of the results each.
template <typename T, int KW, bool OUT, bool REV, bool BWD, bool DOTS> __device__ __forceinline__ void walk_state(const Walk& a, const Role& ro, const Task& k, char* lds) {
  typedef Form<T> F;
  typedef typename F::Frag Frag;
  typedef Cells<T, KW> XC;
  typedef Cells<T, SLAB> ZC;
  typedef Room<T, KW, OUT, BWD> R;
  constexpr int C = R::C, NI = R::NI, NJ = R::NJ, NS = KW / F::K, NT = KW / 16, TP = F::TP, NZT = NJ * TP, ZP = parts_of_z<T>(), PP = parts_of_pairs<T>(DOTS), SP = parts_of_state<T>(DOTS);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l16 = lane & 15, g4 = 4 * (lane >> 4), n0 = k.col0 + 16 * wave;
  const Spot& p = k.p;
  const unsigned lds0 = lds_byte_addr(lds);
  // tile i of the state holds rows 16 i + 4 g + r of column n0 + l16
  floatx4 st[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) st[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  const int n = n0 + l16, step_k = ro.turned ? 1 : a.dv, step_n = ro.turned ? a.dv : 1;
  const int64_t state_size = (int64_t)ro.sk * ro.sn;
  if (OUT && ro.init) {
    const float* s = ro.init + ((int64_t)(a.by_slot ? k.slot : p.row) * a.H + k.h) * state_size + (int64_t)n * step_n;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * i + g4 + r < ro.sk && n < ro.sn) st[i][r] = s[(int64_t)(16 * i + g4 + r) * step_k];
  }
  const bool here = n0 + g4 < ro.vw, full = n0 + 16 <= ro.vw;  // this lane's four columns of a result exist; the wave's
  T* op = OUT ? const_cast<T*>(head_of<T>(ro.out, p, k.h)) + n0 : nullptr;
  unsigned row_off[NI];  // tokens are at most 16 MiB apart
#pragma unroll
  for (int t = 0; t < NI; ++t) row_off[t] = (unsigned)((16 * t + l16) * (int)(OUT ? ro.out.st : 0) + g4);
  const T* wp = DOTS ? head_of<T>(ro.w, p, k.h) : nullptr;
  const int w_col = min(n0 + g4, ro.vw - 4);
  const unsigned xa = lds0 + R::XB + R::ZB + XC::rows(lane), ya = lds0 + XC::cols(lane), za = (lds0 + R::XB + ZC::cols(lane)) ^ (sizeof(T) == 2 ? 32 * wave : 64 * wave);
  // the state is there before the loop begins: a wait for it inside would, from the second turn on, be one for the results' stores
#pragma unroll
  for (int i = 0; i < NT; ++i) asm volatile("" : "+v"(st[i]));
  lds_barrier();  // the first chunk's tiles
  lds_barrier();  // its decays
  const int dir = REV ? -C : C;
  int t0 = chunk_at<REV>(k, 0) * C;
  T* ob = op + t0 * (OUT ? ro.out.st : 0);
  const T* wb = wp + t0 * (DOTS ? ro.w.st : 0);
  const int64_t out_step = dir * (OUT ? ro.out.st : 0), w_step = dir * (DOTS ? ro.w.st : 0);
  typename Vec4<T>::V wr[NI];  // a chunk's partners, fetched when those of the chunk before have been used
  const auto partners = [&](int t0) {  // of tokens and columns that do not exist the last ones': what they give is dropped, or 0
    const int last = min(C, p.len - t0) - 1;
#pragma unroll
    for (int t = 0; t < NI; ++t) wr[t] = *reinterpret_cast<const typename Vec4<T>::V*>(wb + min(16 * t + l16, last) * (int)(DOTS ? ro.w.st : 0) + w_col);
    wb += w_step;
  };
  if (DOTS && k.nchunk > 0) partners(t0);
  floatx4 zero = {0.f, 0.f, 0.f, 0.f};  // kept in registers: a constant would be moved into every sum's at every chunk
  asm volatile("" : "+v"(zero));
  for (int it = 0, at = 0; it < k.nchunk; ++it) {
    const int valid = min(C, p.len - t0);
    const float* f = reinterpret_cast<const float*>(lds + R::FACTORS) + 256 * (it & 1);
    const unsigned xr = xa + at, yc = ya + at, zc = za + at;
    const char* pairs = lds + R::PAIRS;
    // What LDS holds is read well ahead of its use: two steps of x, two parts of the pairs, four tiles of y
    Frag zf[NJ], zs[NJ][ZP], x[3][NI], sp[2][SP], pf[2][R::SLOTS], yf[4][NJ];
    floatx4 acc[NI], low[NI], in[NI], cf[NJ][TP];  // low: of the state's lower parts, summed apart so that their sums are not rounded at the whole's
    const auto read_x = [&](int s) {
#pragma unroll
      for (int t = 0; t < NI; ++t) x[s % 3][t] = XC::by_row(xr, 16 * t * XC::ROWB, s);
    };
    const auto pair_block = [&](int t, int j, int part) -> Frag {
      const char* q = pairs + R::block(t, j, REV);
      if constexpr (TP == 2) {
        if (R::half(t, j, REV)) {
          const bf16x4 there = *reinterpret_cast<const bf16x4*>(q + 512 * part + 8 * lane), none = {};
          return REV ? Mma16::join(none, there) : Mma16::join(there, none);
        }
      }
      return *reinterpret_cast<const Frag*>(q + 1024 * part + 16 * lane);
    };
    const auto read_pairs = [&](int part) {
#pragma unroll
      for (int t = 0; t < NI; ++t)
#pragma unroll
        for (int j = 0; j < NJ; ++j)
          if (R::needed(t, j, REV)) pf[part % 2][R::slot(t, j, REV)] = pair_block(t, j, part);
    };
    const auto read_y = [&](int i) {
#pragma unroll
      for (int j = 0; j < NJ; ++j) yf[i & 3][j] = XC::by_col(yc, F::K * j, i);
    };
    const auto split_state = [&](int s) {
      floatx4 v[TP];
#pragma unroll
      for (int t = 0; t < TP; ++t) v[t] = st[TP * s + t];
      split(v, sp[s & 1]);
    };
    const auto from_state = [&](int s) {  // rows of the result are columns of z, its column is i
#pragma unroll
      for (int part = 0; part < SP; ++part)
#pragma unroll
        for (int t = 0; t < NI; ++t) F::mma(SP == 3 && part ? low[t] : acc[t], sp[s & 1][part], x[s % 3][t]);
    };
    const auto from_pairs = [&] {
#pragma unroll
      for (int part = 0; part < PP; ++part) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int t = 0; t < NI; ++t)
            if (R::needed(t, j, REV)) F::mma(in[t], zf[j], pf[part % 2][R::slot(t, j, REV)]);
        if (part + 2 < PP) read_pairs(part + 2);
      }
    };
    // z with each token's factor, as an operand: one tile
    const auto scaled = [&](auto guard, int j, int t) {
      floatx4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool there = !decltype(guard)::value || F::K * j + 16 * t + g4 + r < valid;  // (0 times what is not finite)
        v[r] = rounded(there ? F::get(zf[j], t, r) * cf[j][t][r] : 0.f);
      }
      if constexpr (TP == 2) {
        bf16x4 part[ZP];
        parts_of(v, part);
#pragma unroll
        for (int i = 0; i < ZP; ++i)
#pragma unroll
          for (int r = 0; r < 4; ++r) zs[j][i][4 * t + r] = part[i][r];
      } else {
        zs[j][0] = v;
      }
    };
    if constexpr (OUT) {
      read_x(0);
      if (NS > 1) read_x(1);
    }
    const float total = f[128];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      zf[j] = ZC::by_col(zc, F::K * j, 0);
#pragma unroll
      for (int t = 0; t < TP; ++t) cf[j][t] = load4(f + 64 + F::K * j + 16 * t + g4);
    }
    __builtin_amdgcn_sched_barrier(0);
    bool fine = true;
#pragma unroll
    for (int j = 0; j < NJ; ++j) fine = fine && all_finite(zf[j]);
    const bool odd = __any(!fine);
    if constexpr (OUT) {
      // ---- what the state gives
#pragma unroll
      for (int t = 0; t < NI; ++t) acc[t] = low[t] = in[t] = zero;
      split_state(0);
#pragma unroll
      for (int s = 0; s < NS; ++s) {
        if (s + 2 < NS) read_x(s + 2);
        __builtin_amdgcn_sched_barrier(0);
        if (s + 1 < NS) split_state(s + 1);
#pragma unroll
        for (int i = s * NZT / NS; i < (s + 1) * NZT / NS; ++i) scaled(std::false_type{}, i / TP, i % TP);
        from_state(s);
        interleave<T, SP * NI, 6>();
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NZT; ++i) scaled(std::false_type{}, i / TP, i % TP);
    }
#pragma unroll
    for (int i = 0; i < 4 && i < NT; ++i) read_y(i);
    // ---- what the chunk's pairs give
    if constexpr (OUT) {
      lds_barrier();
      read_pairs(0);
      if (PP > 1) read_pairs(1);
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < NT; ++i) st[i] *= total;
    if constexpr (OUT) from_pairs();
    if (__builtin_expect(odd, 0)) {
#pragma unroll
      for (int i = 0; i < NZT; ++i) scaled(std::true_type{}, i / TP, i % TP);
      if constexpr (OUT) {
        // A masked pair would be 0 times such a value: they are taken out of the product and added pair by pair
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int t = 0; t < TP; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!is_finite(F::get(zf[j], t, r))) F::put(zf[j], t, r, 0.f);
#pragma unroll
        for (int t = 0; t < NI; ++t) {
          in[t] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int part = 0; part < PP; ++part)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
              if (R::needed(t, j, REV)) F::mma(in[t], zf[j], pair_block(t, j, part));
        }
        const T* zp = head_of<T>(ro.z, p, k.h) + n0 + g4;
#pragma unroll 1
        for (int j = 0; j < valid; ++j) {
          const floatx4 z = here ? load4(zp + (int64_t)(t0 + j) * ro.z.st) : floatx4{0.f, 0.f, 0.f, 0.f};
          const int e = j % 4, tile = j % F::K / 16, from = j % 16 / 4;  // its slot and the lane group that holds it
#pragma unroll
          for (int t = 0; t < NI; ++t) {
            const int i = 16 * t + l16;
            if (REV ? j < i : j > i) continue;
            const bool half = R::half(t, j / F::K, REV);
            const T* q = reinterpret_cast<const T*>(pairs + R::block(t, j / F::K, REV) + (half ? 8 : 16) * (16 * from + l16)) + (half ? 0 : 4 * tile) + e;
            float w = 0.f;
#pragma unroll
            for (int part = 0; part < PP; ++part) w += to_f32(q[part * (half ? 512 : 1024) / sizeof(T)]);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (!is_finite(z[r])) in[t][r] += w * z[r];
          }
        }
      }
    }
    // ---- the state behind the chunk, and beside its products the results
    float rf[NI];
    if constexpr (OUT)
#pragma unroll
      for (int t = 0; t < NI; ++t) rf[t] = f[16 * t + l16];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int part = 0; part < ZP; ++part)
#pragma unroll
        for (int j = 0; j < NJ; ++j) F::mma(st[i], yf[i & 3][j], zs[j][part]);
      if (i + 4 < NT) read_y(i + 4);
    }
    if constexpr (OUT) {
      float d[2 * NI];  // what w makes of them: by the state, by the pairs
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        if (SP == 3) acc[t] += low[t];
        acc[t] *= rf[t];
        if constexpr (DOTS) {
          d[t] = d[NI + t] = 0.f;
#pragma unroll
          for (int r = 0; r < 4; ++r) d[t] += acc[t][r] * to_f32(wr[t][r]), d[NI + t] += in[t][r] * to_f32(wr[t][r]);
        }
        acc[t] += in[t] * a.scale;
      }
      // (the partners are used up before the stores go out: a wait for them behind would be one for the stores)
      if constexpr (DOTS)
#pragma unroll
        for (int t = 0; t < 2 * NI; ++t) asm volatile("" : "+v"(d[t]));
      if (valid == C && full) {
#pragma unroll
        for (int t = 0; t < NI; ++t) store4(ob + row_off[t], acc[t]);
      } else {
#pragma unroll
        for (int t = 0; t < NI; ++t)
          if (16 * t + l16 < valid && here) store4(ob + row_off[t], acc[t]);
      }
      if constexpr (DOTS) {
        // over the lanes of a token: an exchange of two sums leaves one, whose rows of 16 lanes are the first's and the second's in turn
        float* q = reinterpret_cast<float*>(lds + R::DOTS) + (it & 1) * 8 * C + 2 * wave * C;  // [it & 1][wave][inter, pairs][C]
        const int row = lane >> 4;
        if constexpr (NI == 4) {
          float e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) e[i] = rows_join16(d[2 * i], d[2 * i + 1]);  // row r: of d[2 i + r % 2], half r / 2
          const float s0 = rows_join32(e[0], e[1]), s1 = rows_join32(e[2], e[3]);  // row r: of d[2 (r / 2) + r % 2] and four further on
          q[16 * row + l16] = s0;
          q[C + 16 * row + l16] = s1 * a.scale;
        } else {
#pragma unroll
          for (int t = 0; t < NI; ++t) {
            const float s0 = xor32_sum(rows_join16(d[t], d[NI + t]));  // even rows: by the state, odd ones: by the pairs
            if (row < 2) q[row * C + 16 * t + l16] = row ? s0 * a.scale : s0;
          }
        }
      }
    }
    ob += out_step;
    t0 += dir;
    if (DOTS && it + 1 < k.nchunk) partners(t0);
    lds_barrier();
    at = at == (R::RING - 1) * R::BUF ? 0 : at + R::BUF;
  }
  if (ro.fin && (!OUT || (REV ? p.first : p.last))) {
    float* s = ro.fin + ((int64_t)(OUT ? p.row : k.slot) * a.H + k.h) * state_size + (int64_t)n * step_n;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (16 * i + g4 + r < ro.sk && n < ro.sn) s[(int64_t)(16 * i + g4 + r) * step_k] = st[i][r];
  }
}

template <typename T, int KW, bool OUT, bool BWD> __global__ __launch_bounds__(WALK_THREADS) void decay_walk_kernel(Walk a) {
  typedef Room<T, KW, OUT, BWD> R;
  extern __shared__ __attribute__((aligned(1024))) char lds[];
  // workgroups of one (slot, head) follow each other on one XCD, whose L2 then holds what they share
  const int w = blockIdx.x;
  int unit, item;
  if (a.units % 8 == 0) {
    unit = (w >> 3) / a.per * 8 + (w & 7);
    item = (w >> 3) % a.per;
  } else {
    unit = w / a.per;
    item = w % a.per;
  }
  int which = 0;
  while (item >= a.role[which].slabs) item -= a.role[which++].slabs;
  const Role& ro = a.role[which];
  Task k;
  k.slot = unit / a.H, k.h = unit % a.H, k.item = item;
  k.p = spot(a, k.slot);
  if (!k.p.on) return;
  if (!OUT && (ro.rev ? k.p.first : k.p.last)) return;  // nothing walks on from there
  k.nchunk = (k.p.len + R::C - 1) / R::C, k.col0 = item * SLAB, k.vw = min(SLAB, ro.vw - k.col0);
  if (ro.kw < KW || k.vw < SLAB) {
    for (int i = threadIdx.x * 16; i < R::PAIRS; i += WALK_THREADS * 16) *reinterpret_cast<floatx4*>(lds + i) = floatx4{0.f, 0.f, 0.f, 0.f};
    lds_barrier();
  }
  if (threadIdx.x >= 256) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - 4;
    if (ro.rev) pair_wave<T, KW, OUT, true, BWD>(wave, a, ro, k, lds);
    else pair_wave<T, KW, OUT, false, BWD>(wave, a, ro, k, lds);
  } else if (BWD && ro.dots) {
    if (ro.rev) walk_state<T, KW, OUT, true, BWD, BWD>(a, ro, k, lds);
    else walk_state<T, KW, OUT, false, BWD, BWD>(a, ro, k, lds);
  } else {
    if (ro.rev) walk_state<T, KW, OUT, true, BWD, false>(a, ro, k, lds);
    else walk_state<T, KW, OUT, false, BWD, false>(a, ro, k, lds);
  }
}

// States before every segment (behind it, backwards) from what each adds: in place, four elements a thread, a row's segments one after the other.
struct Join {
  float* states;
  const float *whole, *init;
  const int32_t* cu;
  int H, T, nseq, seg, nseg, rev;
  int64_t size;
};
__global__ __launch_bounds__(JOIN_THREADS) void decay_join_kernel(Join a) {
  const int row = blockIdx.x / a.H, h = blockIdx.x % a.H;
  int64_t slot = (int64_t)row * a.nseg;
  int n = a.nseg;
  if (a.nseq) {
    const int from = seq_first(a.cu, row, a.T), len = seq_end(a.cu, row, a.T) - from;
    n = max(1, (int)(((unsigned)len + a.seg - 1) / a.seg));
    slot = packed_slot(from, row, a.seg);
  }
  const int64_t e0 = ((int64_t)blockIdx.y * JOIN_THREADS + threadIdx.x) * 4;
  const int many = (int)min((int64_t)4, a.size - e0);
  constexpr int U = 4;  // segments fetched together
  float s[4], add[U][4], f[U];
  const auto segment = [&](int i) { return slot + (a.rev ? n - 1 - i : i); };
  const auto get = [&](float (&x)[4], const float* q) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = q && e < many ? q[e] : 0.f;
  };
  get(s, a.init ? a.init + ((int64_t)row * a.H + h) * a.size + e0 : nullptr);
  for (int i0 = 0; i0 < n; i0 += U) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const bool on = i0 + u + 1 < n;  // nothing walks on from the last one, which left nothing
      const int64_t at = on ? segment(i0 + u) * a.H + h : 0;
      get(add[u], on ? a.states + at * a.size + e0 : nullptr);
      f[u] = on ? a.whole[at] : 0.f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u >= n) break;
      float* q = a.states + (segment(i0 + u) * a.H + h) * a.size + e0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (e < many) q[e] = s[e];
        s[e] = f[u] * s[e] + add[u][e];
      }
    }
  }
}

// Sums over C lanes, in every one of them
template <int CTRL> __device__ __forceinline__ double from_lane64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint64_t lo = (unsigned)__builtin_amdgcn_mov_dpp((int)u, CTRL, 0xF, 0xF, true), hi = (unsigned)__builtin_amdgcn_mov_dpp((int)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, hi << 32 | lo);
}
template <int C> __device__ __forceinline__ float chunk_sum(float x) {
  x = row16_sum(x);
  if constexpr (C >= 32) x = xor16_sum(x);
  if constexpr (C == 64) x = xor32_sum(x);
  return x;
}
template <int C> __device__ __forceinline__ double chunk_sum(double x) {
  x += from_lane64<0xB1>(x);
  x += from_lane64<0x4E>(x);
  x += from_lane64<0x141>(x);
  x += from_lane64<0x128>(x);
  const auto both = [](uint64_t lo, uint64_t hi) { return __builtin_bit_cast(double, hi << 32 | (unsigned)lo); };
  if constexpr (C >= 32) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = __builtin_amdgcn_permlane16_swap((unsigned)u, (unsigned)u, false, false), hi = __builtin_amdgcn_permlane16_swap((unsigned)(u >> 32), (unsigned)(u >> 32), false, false);
    x = both(lo[0], hi[0]) + both(lo[1], hi[1]);
  }
  if constexpr (C == 64) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = __builtin_amdgcn_permlane32_swap((unsigned)u, (unsigned)u, false, false), hi = __builtin_amdgcn_permlane32_swap((unsigned)(u >> 32), (unsigned)(u >> 32), false, false);
    x = both(lo[0], hi[0]) + both(lo[1], hi[1]);
  }
  return x;
}

// dg from the walks' dots.  In a chunk with W = <dS, S> behind it:
//   dg_t = sum_{s >= t} (x_s + u_s) + sum_{r < t} y_r + Z     Z = W - sum y     W before the chunk = Z + sum x
// x: what a token's outputs took from the state before the chunk, y: what its key hands to the state behind it, u: its pairs as a query less those as
// a key.  A strong decay makes x, y and Z small, and they are summed apart from the pairs, which cancel over a chunk.
// W is known at both ends of a segment, from the states there.  Walked from its end the sums miss it at its beginning by what their terms were off, which
// for a slow decay is a drift; that is taken back from the chunks in the proportion of sum |x| + |y| (H8 T4096 d128: dg off by 1.1e-6 -> 2.2e-7 against 64 bits),
// so that a quiet part of a row has no share in what a loud one is off by (H130 T4096 d64, the half of a row whose other half's values are a thousand times its own:
// 2e-4 - 1.6e-3 of its norm if evenly, at most 3e-6 thus; the kernel 21.0 us -> 22.2 at B8 H16 T4096 d128).  A chunk's sum is of the same differences as the row's, in double.
// Where a term is not finite the sums from the end are not either, from its token down; a key's or a value's leaves its own dg and the earlier ones be,
// which then come from the segment's beginning:
//   dg_t = sum_{r < t} (y_r - x_r - u_r) + W before the chunk     W behind the chunk = W before + sum (y - x)
struct GateGrad {
  const float *dots_q, *dots_k;  // [inter, pairs][slab][B H][T]
  const float *init, *d_init, *fin, *d_fin;  // of rows, or NULL
  const float *before, *behind;  // of segments: the state before each, the state's gradient behind it
  const int32_t* cu;
  float *dg, *part;  // part: sums over a segment, [slot][H]
  int B, H, T, nseq, slabs, seg, nseg;
  int64_t step, size;
};
template <int C> __global__ __launch_bounds__(GATE_THREADS) void decay_gate_grad_kernel(GateGrad a) {
  constexpr int NC = GATE_THREADS / C, U = 4;  // chunks of a turn; turns whose dots are fetched together
  __shared__ double chunk[2][NC], red[16];
  const int slot = blockIdx.x / a.H, h = blockIdx.x % a.H, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, in = lane % C, mine = threadIdx.x / C;
  const Spot p = spot(a, slot);
  if (!p.on) {
    if (a.part && threadIdx.x == 0) a.part[(int64_t)slot * a.H + h] = 0.f;
    return;
  }
  const int len = p.len;
  const int64_t base = (int64_t)(p.b * a.H + h) * a.T + p.tok;
  const auto block_sum = [&](double x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o, LNX_WAVE);
    __syncthreads();
    if (lane == 0) red[wave] = x;
    __syncthreads();
    double s = 0.;
    for (int i = 0; i < 16; ++i) s += red[i];
    return s;
  };
  const auto product = [&](const float* s, const float* d, int64_t i, int64_t j) {  // of two states, this thread's part
    float w = 0.f;
    if (s && d) {
      s += (i * a.H + h) * a.size, d += (j * a.H + h) * a.size;
#pragma unroll 8
      for (int e = threadIdx.x; e < (int)a.size; e += GATE_THREADS) w += s[e] * d[e];
    }
    return (double)w;
  };
  float x[U], y[U], u[U];
  const auto get = [&](int t, float& x, float& y, float& u) {
    x = y = u = 0.f;
    if (t < 0 || t >= len) return;
    for (int s = 0; s < a.slabs; ++s) {
      x += a.dots_q[s * a.step + base + t];
      y += a.dots_k[s * a.step + base + t];
      u += a.dots_q[(a.slabs + s) * a.step + base + t] - a.dots_k[(a.slabs + s) * a.step + base + t];
    }
  };
  const auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < U; ++i) get(t - i * GATE_THREADS, x[i], y[i], u[i]);
  };
  const int top = len > 0 ? (len - 1) / GATE_THREADS * GATE_THREADS + (int)threadIdx.x : (int)threadIdx.x;
  fetch(top);
  double off = 0., loud = 0.;
#pragma unroll
  for (int i = 0; i < U; ++i) off += x[i] - y[i], loud += fabsf(x[i]) + fabsf(y[i]);
  for (int t = top - U * GATE_THREADS; t >= 0; t -= GATE_THREADS) {
    float nx, ny, nu;
    get(t, nx, ny, nu);
    off += nx - ny, loud += fabsf(nx) + fabsf(ny);
  }
  const double end = p.last ? product(a.fin, a.d_fin, p.row, p.row) : product(a.before, a.behind, slot + 1, slot);
  const double begin = p.first ? product(a.init, a.d_init, p.row, p.row) : product(a.before, a.behind, slot, slot - 1);
  double W = block_sum(end);
  off = block_sum(off + end - begin);
  int good = -1;  // tokens up to here: from the beginning
  double B = 0.;
  if (!is_finite((float)off)) {
    off = 0.;
    int bad = len;
    for (int64_t t = threadIdx.x; t < bad; t += GATE_THREADS) {  // (rows may end within GATE_THREADS of 2^31)
      float ax, ay, au;
      get((int)t, ax, ay, au);
      if (!is_finite(ax + ay + au)) bad = (int)t;
    }
    B = block_sum(begin);
#pragma unroll
    for (int o = 32; o; o >>= 1) bad = min(bad, __shfl_xor(bad, o, LNX_WAVE));
    __syncthreads();
    if (lane == 0) red[wave] = bad;
    __syncthreads();
    for (int i = 0; i < 16; ++i) bad = min(bad, (int)red[i]);
    if (is_finite((float)B)) good = min(bad, len - 1);
  }
  loud = block_sum(loud);
  const double drift = loud > 0. && off != 0. ? off / loud : 0.;
  double sum = 0.;
  for (int t = top, turn = 0; t - (int)threadIdx.x >= 0 || turn == 0; t -= U * GATE_THREADS) {
    if (turn) fetch(t);
#pragma unroll
    for (int i = 0; i < U; ++i, ++turn) {
      const int ti = t - i * GATE_THREADS;
      if (ti - (int)threadIdx.x < 0) break;  // (of the workgroup)
      float sx = x[i], su = u[i], py = y[i];
#pragma unroll
      for (int o = 1; o < C; o <<= 1) {
        const float bx = __shfl_down(sx, o, LNX_WAVE), bu = __shfl_down(su, o, LNX_WAVE), by = __shfl_up(py, o, LNX_WAVE);
        if (in + o < C) sx += bx, su += bu;
        if (in >= o) py += by;
      }
      const float Y = __shfl(py, lane - in + C - 1, LNX_WAVE);
      const double step = chunk_sum<C>((double)(x[i] - y[i]));  // as the sum over the row took them
      const float weight = chunk_sum<C>(fabsf(x[i]) + fabsf(y[i]));
      if (in == 0) chunk[turn & 1][mine] = step - weight * drift;
      __syncthreads();
      double behind = W;
#pragma unroll 8
      for (int j = NC - 1; j >= 0; --j) {
        if (j == mine) behind = W;
        W += chunk[turn & 1][j];
      }
      const float Z = (float)(behind - Y);
      const float d = sx + su + (py - y[i]) + Z;
      if (ti < len && ti > good) {
        if (a.dg) a.dg[base + ti] = d;
        sum += d;
      }
    }
  }
  __syncthreads();
  int turn = 0;
  for (int64_t t = threadIdx.x; t - (int)threadIdx.x <= good; t += GATE_THREADS, ++turn) {
    float ax, ay, au;
    get(t < good ? (int)t : -1, ax, ay, au);
    const float own = ay - ax - au;
    float before = own, all = ay - ax;
#pragma unroll
    for (int o = 1; o < C; o <<= 1) {
      const float bb = __shfl_up(before, o, LNX_WAVE), ba = __shfl_up(all, o, LNX_WAVE);
      if (in >= o) before += bb, all += ba;
    }
    if (in == C - 1) chunk[turn & 1][mine] = all;
    __syncthreads();
    double from = B;
#pragma unroll 8
    for (int j = 0; j < NC; ++j) {
      if (j == mine) from = B;
      B += chunk[turn & 1][j];
    }
    if (t <= good) {
      const float d = (float)from + (before - own);
      if (a.dg) a.dg[base + t] = d;
      sum += d;
    }
  }
  if (a.part) {
    const double s = block_sum(sum);
    if (threadIdx.x == 0) a.part[(int64_t)slot * a.H + h] = (float)s;
  }
}
// dg[h] = sum of the segments' sums
__global__ __launch_bounds__(256) void decay_gate_sum_kernel(const float* part, int64_t rows, int H, float* dg) {
  __shared__ float red[4];
  float s = 0.f;
  for (int64_t r = threadIdx.x; r < rows; r += 256) s += part[r * H + blockIdx.x];
  s = wave_sum(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) dg[blockIdx.x] = (red[0] + red[1]) + (red[2] + red[3]);
}

// One token: a workgroup per (row, head, 128 columns).  Bound by the state, read and written once.
struct Step {
  const void *q, *k, *v;
  const float *g, *s0;
  void* o;
  float* s1;
  int64_t gb, gh;
  int H, dk, dv, slabs;
  float scale;
};
constexpr int STEP_COLS = 128, STEP_MAX_DK = 256;
template <typename T, int VN> __global__ __launch_bounds__(STEP_THREADS) void decay_step_kernel(Step a) {
  constexpr int LPR = STEP_COLS / VN, GROUPS = STEP_THREADS / LPR, U = 8;  // lanes of a row, rows at a time
  __shared__ float qk[2][STEP_MAX_DK], red[GROUPS][STEP_COLS];
  const int slab = blockIdx.x % a.slabs, bh = blockIdx.x / a.slabs, h = bh % a.H, li = threadIdx.x % LPR, grp = threadIdx.x / LPR, c = slab * STEP_COLS + li * VN;
  const float f = __expf(a.g[bh / a.H * a.gb + h * a.gh]);
  for (int i = threadIdx.x; i < a.dk; i += STEP_THREADS) {
    qk[0][i] = to_f32(static_cast<const T*>(a.q)[(int64_t)bh * a.dk + i]) * a.scale;
    qk[1][i] = to_f32(static_cast<const T*>(a.k)[(int64_t)bh * a.dk + i]);
  }
  float v[VN], o[VN];
#pragma unroll
  for (int e = 0; e < VN; ++e) {
    v[e] = c + e < a.dv ? to_f32(static_cast<const T*>(a.v)[(int64_t)bh * a.dv + c + e]) : 0.f;
    o[e] = 0.f;
  }
  __syncthreads();
  const int64_t base = (int64_t)bh * a.dk * a.dv + c;
  for (int i0 = grp; i0 < a.dk; i0 += GROUPS * U) {
    float s[U][VN];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * GROUPS;
      const float* p = a.s0 + base + (int64_t)i * a.dv;
      if constexpr (VN == 4) {
        floatx4 x = {0.f, 0.f, 0.f, 0.f};
        if (i < a.dk && c < a.dv) x = load4(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) s[u][e] = x[e];
      } else {
        s[u][0] = i < a.dk && c < a.dv ? p[0] : 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * GROUPS;
      if (i >= a.dk || c >= a.dv) continue;
      const float qi = qk[0][i], ki = qk[1][i];
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        s[u][e] = f * s[u][e] + ki * v[e];
        o[e] += qi * s[u][e];
      }
      float* p = a.s1 + base + (int64_t)i * a.dv;
      if constexpr (VN == 4) store4(p, floatx4{s[u][0], s[u][1], s[u][2], s[u][3]});
      else p[0] = s[u][0];
    }
  }
#pragma unroll
  for (int e = 0; e < VN; ++e) red[grp][li * VN + e] = o[e];
  __syncthreads();
  const int col = slab * STEP_COLS + threadIdx.x;
  if (threadIdx.x < STEP_COLS && col < a.dv) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) s += red[i][threadIdx.x];
    static_cast<T*>(a.o)[(int64_t)bh * a.dv + col] = from_f32<T>(s);
  }
}

// ---------------------------------------------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------------------------------------------

int up(int x, int to) { return (x + to - 1) / to * to; }
int64_t ceil_div(int64_t x, int64_t y) { return (x + y - 1) / y; }
constexpr int MAX_D = 256;

// Tokens of a segment, a multiple of 64, or 0: rows are walked whole.  Segments read keys and values (queries and gradients) once more, so they
// are for rows and heads that leave CUs without a workgroup: as many as give every CU one (H16 T65000 d128, with two bf16 parts of what a token adds: 290 us
// and 125 on the local walks, with two a CU 310 and 138; with three parts 306 and 147), of four chunks and more, for rows of more than eight (us of forward alone and with backward, chunks of 64, eight and
// more -> four: H8 T1000 d128 35, 79 -> 27, 62; H16 T700 34, 77 -> 25, 68; of two 25, 70 and 23, 74; H16 T500 d64 whole 15, 37, in two 20, 45).
// The rows of a packed batch are taken for one: their lengths are not known here, and sequences of one segment are walked once whatever its size.
int segment(const lnx_decay_args* a) {
  const int64_t walks = (a->nseq ? 1 : (int64_t)a->B) * a->H * ceil_div(a->dv, SLAB);
  const int shortest = a->dtype == LNX_BF16 ? 256 : 128;
  if (walks > 128 || a->T <= 2 * shortest) return 0;
  const int s = up((int)ceil_div(a->T, 256 / walks), 64);
  return s < shortest ? shortest : s >= a->T ? 0 : s;
}
struct Layout {
  int seg, nseg;
  int64_t slots, rows;
  int64_t states, factors, dots, part, d_init;  // bytes: states of all segments, their factors, the walks' dots, segments' sums, gradients of the initial states that the caller does not want
};
Layout layout(const lnx_decay_args* a) {
  Layout l{};
  const int s = segment(a);
  l.rows = a->nseq ? a->nseq : a->B;
  l.seg = s ? s : 0x7fffffc0;
  l.nseg = s ? (int)ceil_div(a->T, s) : 1;
  l.slots = a->nseq ? a->T / l.seg + a->nseq : (int64_t)a->B * l.nseg;
  if (s) l.states = l.slots * a->H * a->dk * a->dv * 4, l.factors = ceil_div(l.slots * a->H * 4, 16) * 16;
  l.dots = ceil_div(4 * ceil_div(a->dk, SLAB) * a->B * a->H * (int64_t)a->T * 4, 16) * 16;
  l.part = l.slots * a->H * 4;
  if (a->initial_state && !a->d_initial_state) l.d_init = l.rows * a->H * a->dk * a->dv * 4;
  return l;
}

bool aligned(const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int check(const char* what, const lnx_decay_args* a, bool bwd) {
  if (!a) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (a->B < 0 || a->H <= 0 || a->T < 0 || a->T > 0x7fffff00 || a->dk <= 0 || a->dk > MAX_D || a->dv <= 0 || a->dv > MAX_D || a->nseq < 0 || (a->nseq && a->B != 1))
    return lnx_set_error(LNX_ERR_SHAPE, "%s: unsupported dimensions B=%d H=%d T=%d dk=%d dv=%d nseq=%d (heads of at most %d; packed batches have B = 1)", what, a->B, a->H, a->T,
                         a->dk, a->dv, a->nseq, MAX_D);
  if (a->dtype != LNX_F32 && a->dtype != LNX_BF16) return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return lnx_set_error(LNX_ERR_SHAPE, "%s: scale must be finite", what);
  if (a->nseq && !a->cu_seqlens) return lnx_set_error(LNX_ERR_NULL, "%s: nseq without cu_seqlens", what);
  if (bwd && a->g_per_head) {  // written whether there are rows or not
    if (!a->d_g) return lnx_set_error(LNX_ERR_NULL, "%s: d_g is required", what);
    if (a->H > MAX_GRID / 256) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many heads", what);
  }
  if (a->B == 0) return LNX_OK;
  const Layout l = layout(a);
  const int64_t walks = l.slots * a->H * (bwd ? 2 * ceil_div(a->dk, SLAB) + ceil_div(a->dv, SLAB) : ceil_div(a->dv, SLAB));
  if (walks > MAX_GRID / WALK_THREADS || (bwd ? l.slots * a->H > MAX_GRID / GATE_THREADS : l.rows * a->H > MAX_GRID / JOIN_THREADS)) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  if (!bwd && !a->final_state) return lnx_set_error(LNX_ERR_NULL, "%s: final_state is required", what);
  if (bwd && a->d_final_state && !a->final_state) return lnx_set_error(LNX_ERR_NULL, "%s: d_final_state needs final_state", what);
  if (bwd && a->T && !a->d_g) return lnx_set_error(LNX_ERR_NULL, "%s: d_g is required", what);
  const lnx_tensor4* ts[] = {&a->q, &a->k, &a->v, &a->o, &a->d_o, &a->d_q, &a->d_k, &a->d_v};
  const int64_t size = a->dtype == LNX_BF16 ? 2 : 4;
  const auto fits = [&](int extent, int64_t stride) { return extent <= 1 || stride * size % 16 == 0; };
  for (int i = 0; i < 8; ++i) {
    if (bwd ? i == 3 : i > 3) continue;
    const lnx_tensor4& t = *ts[i];
    if (a->T && !t.p) return lnx_set_error(LNX_ERR_NULL, "%s: a tensor is missing", what);
    if (!aligned(t.p, 16) || !fits(a->B, t.stride_b) || !fits(a->H, t.stride_h) || !fits(a->T, t.stride_t) || (a->T > 1 && (t.stride_t < 0 || t.stride_t * size > 1 << 24)))
      return lnx_set_error(LNX_ERR_SHAPE, "%s: tensors must be 16-byte aligned, rows whole numbers of 16 bytes and at most 16 MiB apart", what);
  }
  if (a->T && !a->g) return lnx_set_error(LNX_ERR_NULL, "%s: g is required", what);
  if (bwd && l.states && !a->kept) return lnx_set_error(LNX_ERR_NULL, "%s: needs what the forward call kept", what);
  const uint64_t need = bwd ? lnx_decay_bwd_workspace_bytes(a) : lnx_decay_fwd_workspace_bytes(a);
  if (need && (!a->workspace || a->workspace_bytes < need || !aligned(a->workspace, 16)))
    return lnx_set_error(LNX_ERR_WORKSPACE, "%s: needs a 16-byte aligned workspace of %llu bytes", what, (unsigned long long)need);
  return LNX_OK;
}

Side side(const lnx_decay_args* a, const lnx_tensor4& t) {
  return {t.p, a->B > 1 ? t.stride_b : 0, a->H > 1 ? t.stride_h : 0, a->T > 1 ? t.stride_t : 0};
}
int width(const lnx_decay_args* a, int d) { return up(d, a->dtype == LNX_BF16 ? 8 : 4); }

// dims: of y in the state and of z
Role role(const lnx_decay_args* a, const lnx_tensor4& x, const lnx_tensor4& y, const lnx_tensor4& z, const lnx_tensor4& out, int sk, int sn, bool rev, bool turned) {
  Role r{};
  r.x = side(a, x), r.y = side(a, y), r.z = side(a, z), r.out = side(a, out);
  r.sk = sk, r.sn = sn, r.kw = width(a, sk), r.vw = width(a, sn);
  r.rev = rev, r.turned = turned, r.slabs = (int)ceil_div(sn, SLAB);
  r.row_scale = rev ? 1.f : a->scale, r.col_scale = rev ? a->scale : 1.f;
  return r;
}
Walk walk(const lnx_decay_args* a, const Layout& l) {
  Walk k{};
  k.g = a->g, k.gb = a->B > 1 ? a->g_stride_b : 0, k.gh = a->H > 1 ? a->g_stride_h : 0, k.gt = a->T > 1 ? a->g_stride_t : 0;
  k.cu = a->cu_seqlens;
  k.B = a->B, k.H = a->H, k.T = a->T, k.nseq = a->nseq, k.dv = a->dv, k.seg = l.seg, k.nseg = l.nseg, k.by_slot = l.states != 0;
  k.units = (int)(l.slots * a->H), k.scale = a->scale;
  k.dots_step = (int64_t)a->B * a->H * a->T;
  return k;
}

template <typename T, int KW, bool OUT, bool BWD> int start(const Walk& k, const char* name, hipStream_t st) {
  const auto kernel = decay_walk_kernel<T, KW, OUT, BWD>;
  constexpr int bytes = Room<T, KW, OUT, BWD>::BYTES;
  static_assert(bytes <= 160 * 1024, "LDS of a CU");
  if (int rc = lnx_lds_limit(reinterpret_cast<const void*>(kernel), bytes)) return rc;
  lnx_profile_mark(name, st);
  hipLaunchKernelGGL(kernel, dim3((unsigned)((int64_t)k.units * k.per)), dim3(WALK_THREADS), bytes, st, k);
  return LNX_OK;
}
template <typename T, bool OUT, bool BWD> int start(Walk& k, int roles, const char* name, hipStream_t st) {
  k.per = 0;
  int kw = 0;  // the widest of the launch's keys
  for (int i = 0; i < roles; ++i) k.per += k.role[i].slabs, kw = kw < k.role[i].kw ? k.role[i].kw : kw;
  if (kw <= 64) return start<T, 64, OUT, BWD>(k, name, st);
  if (kw <= 128) return start<T, 128, OUT, BWD>(k, name, st);
  return start<T, 256, OUT, BWD>(k, name, st);
}

void join(const lnx_decay_args* a, const Layout& l, float* states, const float* whole, const float* init, bool rev, hipStream_t st) {
  Join j{states, whole, init, a->cu_seqlens, a->H, a->T, a->nseq, l.seg, l.nseg, rev, (int64_t)a->dk * a->dv};
  lnx_profile_mark("decay_join", st);
  decay_join_kernel<<<dim3((unsigned)(l.rows * a->H), (unsigned)ceil_div(j.size, 4 * JOIN_THREADS)), JOIN_THREADS, 0, st>>>(j);
}

template <typename T> int forward(const lnx_decay_args* a, hipStream_t st) {
  const Layout l = layout(a);
  Walk k = walk(a, l);
  Role r = role(a, a->q, a->k, a->v, a->o, a->dk, a->dv, false, false);
  r.init = a->initial_state;
  if (l.states) {
    char* ws = static_cast<char*>(a->workspace);
    float* states = a->kept ? a->kept : reinterpret_cast<float*>(ws + l.factors);
    k.whole = reinterpret_cast<float*>(ws);
    k.role[0] = r;
    k.role[0].fin = states;
    if (int rc = start<T, false, false>(k, 1, "decay_local", st)) return rc;
    join(a, l, states, k.whole, a->initial_state, false, st);
    r.init = states;
  }
  r.fin = a->final_state;
  k.role[0] = r;
  return start<T, true, false>(k, 1, "decay_fwd", st);
}

void gate_sum(const lnx_decay_args* a, const float* part, int64_t rows, hipStream_t st) {
  lnx_profile_mark("decay_gate_sum", st);
  decay_gate_sum_kernel<<<dim3((unsigned)a->H), 256, 0, st>>>(part, rows, a->H, a->d_g);
}

template <typename T> int backward(const lnx_decay_args* a, hipStream_t st) {
  const Layout l = layout(a);
  Walk k = walk(a, l);
  char* ws = static_cast<char*>(a->workspace);
  Role q = role(a, a->d_o, a->v, a->k, a->d_q, a->dv, a->dk, false, true), kk = role(a, a->v, a->d_o, a->q, a->d_k, a->dv, a->dk, true, true),
       v = role(a, a->k, a->q, a->d_o, a->d_v, a->dk, a->dv, true, false);
  q.w = side(a, a->q), kk.w = side(a, a->k);
  q.dots = reinterpret_cast<float*>(ws), kk.dots = q.dots + 2 * q.slabs * k.dots_step;
  q.init = l.states ? a->kept : a->initial_state;
  kk.init = v.init = a->d_final_state;
  int64_t at = ceil_div(l.dots + l.part, 16) * 16;
  float* states = nullptr;
  if (l.states) {
    k.whole = reinterpret_cast<float*>(ws + at), at += l.factors;
    states = reinterpret_cast<float*>(ws + at), at += l.states;
    k.role[0] = v;
    k.role[0].fin = states;
    if (int rc = start<T, false, false>(k, 1, "decay_local", st)) return rc;
    join(a, l, states, k.whole, a->d_final_state, true, st);
    kk.init = v.init = states;
  }
  v.fin = l.d_init ? reinterpret_cast<float*>(ws + at) : a->d_initial_state;
  const int wide = a->dk > a->dv ? a->dk : a->dv, narrow = a->dk + a->dv - wide;
  const auto step = [](int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; };
  k.role[0] = q, k.role[1] = kk, k.role[2] = v;
  if (step(wide) == step(narrow)) {
    if (int rc = start<T, true, true>(k, 3, "decay_bwd", st)) return rc;
  } else {
    if (int rc = start<T, true, true>(k, 2, "decay_bwd_qk", st)) return rc;
    k.role[0] = v;
    if (int rc = start<T, true, false>(k, 1, "decay_bwd_v", st)) return rc;
  }
  GateGrad d{};
  d.dots_q = q.dots, d.dots_k = kk.dots, d.init = a->initial_state, d.d_init = v.fin, d.fin = a->final_state, d.d_fin = a->d_final_state, d.cu = a->cu_seqlens;
  d.before = a->kept, d.behind = states, d.seg = l.seg, d.nseg = l.nseg;
  if (a->g_per_head) d.part = reinterpret_cast<float*>(ws + l.dots);
  else d.dg = a->d_g;
  d.B = a->B, d.H = a->H, d.T = a->T, d.nseq = a->nseq, d.slabs = q.slabs, d.step = k.dots_step, d.size = (int64_t)a->dk * a->dv;
  lnx_profile_mark("decay_gate_grad", st);
  const dim3 grid((unsigned)(l.slots * a->H));
  if (q.kw <= 128) decay_gate_grad_kernel<chunk_of<T, 128>()><<<grid, GATE_THREADS, 0, st>>>(d);
  else decay_gate_grad_kernel<chunk_of<T, 256>()><<<grid, GATE_THREADS, 0, st>>>(d);
  if (a->g_per_head) gate_sum(a, d.part, l.slots, st);
  return LNX_OK;
}

int finish(const char* what, int rc, hipStream_t st) {
  if (rc) return rc;
  lnx_profile_mark(nullptr, st);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? LNX_OK : lnx_set_error(LNX_ERR_LAUNCH, "%s: %s", what, hipGetErrorString(e));
}

bool sizes(const lnx_decay_args* a) {
  return a && a->B > 0 && a->H > 0 && a->T >= 0 && a->T <= 0x7fffff00 && a->dk > 0 && a->dk <= MAX_D && a->dv > 0 && a->dv <= MAX_D && a->nseq >= 0;
}

}  // namespace

extern "C" uint64_t lnx_decay_kept_bytes(const lnx_decay_args* a) { return sizes(a) ? layout(a).states : 0; }
extern "C" uint64_t lnx_decay_fwd_workspace_bytes(const lnx_decay_args* a) {
  if (!sizes(a)) return 0;
  const Layout l = layout(a);
  return l.states ? l.factors + (a->kept ? 0 : l.states) : 0;
}
extern "C" uint64_t lnx_decay_bwd_workspace_bytes(const lnx_decay_args* a) {
  if (!sizes(a)) return 0;
  const Layout l = layout(a);
  return ceil_div(l.dots + l.part, 16) * 16 + l.factors + l.states + l.d_init;
}
extern "C" int lnx_decay_fwd(const lnx_decay_args* a, void* hip_stream) {
  if (int rc = check("decay_fwd", a, false)) return rc;
  if (a->B == 0) return LNX_OK;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  return finish("decay_fwd", a->dtype == LNX_BF16 ? forward<bf16_t>(a, st) : forward<float>(a, st), st);
}
extern "C" int lnx_decay_bwd(const lnx_decay_args* a, void* hip_stream) {
  if (int rc = check("decay_bwd", a, true)) return rc;
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  if (a->B == 0) {
    if (!a->g_per_head) return LNX_OK;
    gate_sum(a, nullptr, 0, st);  // sums over no rows are zeros
    return finish("decay_bwd", LNX_OK, st);
  }
  return finish("decay_bwd", a->dtype == LNX_BF16 ? backward<bf16_t>(a, st) : backward<float>(a, st), st);
}
extern "C" int lnx_decay_step(const lnx_decay_step_args* a, void* hip_stream) {
  const char* what = "decay_step";
  if (!a) return lnx_set_error(LNX_ERR_NULL, "%s: args is NULL", what);
  if (a->B < 0 || a->H <= 0 || a->dk <= 0 || a->dk > STEP_MAX_DK || a->dv <= 0)
    return lnx_set_error(LNX_ERR_SHAPE, "%s: unsupported dimensions B=%d H=%d dk=%d dv=%d (dk at most %d)", what, a->B, a->H, a->dk, a->dv, STEP_MAX_DK);
  if (a->dtype != LNX_F32 && a->dtype != LNX_BF16) return lnx_set_error(LNX_ERR_DTYPE, "%s: dtype %d", what, a->dtype);
  if (!(a->scale == a->scale) || a->scale - a->scale != 0.f) return lnx_set_error(LNX_ERR_SHAPE, "%s: scale must be finite", what);
  if (a->B == 0) return LNX_OK;
  if (!a->q || !a->k || !a->v || !a->g || !a->state || !a->o || !a->new_state) return lnx_set_error(LNX_ERR_NULL, "%s: a tensor is missing", what);
  Step k{a->q, a->k, a->v, a->g, a->state, a->o, a->new_state, a->B > 1 ? a->g_stride_b : 0, a->H > 1 ? a->g_stride_h : 0, a->H, a->dk, a->dv, (int)ceil_div(a->dv, STEP_COLS), a->scale};
  const int64_t grid = (int64_t)a->B * a->H * k.slabs;
  if (grid > MAX_GRID / STEP_THREADS) return lnx_set_error(LNX_ERR_SHAPE, "%s: too many rows", what);
  const bool vec = a->dv % 4 == 0 && aligned(a->state, 16) && aligned(a->new_state, 16);
  hipStream_t st = static_cast<hipStream_t>(hip_stream);
  lnx_profile_mark(what, st);
  if (a->dtype == LNX_BF16) {
    if (vec) decay_step_kernel<bf16_t, 4><<<dim3((unsigned)grid), STEP_THREADS, 0, st>>>(k);
    else decay_step_kernel<bf16_t, 1><<<dim3((unsigned)grid), STEP_THREADS, 0, st>>>(k);
  } else {
    if (vec) decay_step_kernel<float, 4><<<dim3((unsigned)grid), STEP_THREADS, 0, st>>>(k);
    else decay_step_kernel<float, 1><<<dim3((unsigned)grid), STEP_THREADS, 0, st>>>(k);
  }
  return finish(what, LNX_OK, st);
}
