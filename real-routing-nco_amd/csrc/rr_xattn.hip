// Cross attention: Lq queries of Hq heads on Lk keys of Hk heads (Hq = G Hk), forward and backward, float32 / float16 / bfloat16.
//
//   s = scale q.k over the visible keys (mask, kv_lens),  p = softmax(s),  o = sum p v,  lse = log sum exp s
//   a row that sees no key: o = 0, lse = -inf, no gradient
//   delta = sum_d do o,  ds = p (do.v - delta),  dq = scale sum ds k,  dk = scale sum ds q,  dv = sum p do   (dk, dv over the group)
//
// Rows: the G Lq queries that share a key head are one list of rows (row = group member * Lq + position), so that a tile of keys
// and values is read once for all of them; with one query a group of heads still fills a matrix tile.
// Tiles: scores are computed transposed, S^T = K Q^T in 16 x 16 tiles, so that a lane holds one query's scores of four consecutive
// keys: the softmax's rescaling is one factor a lane, and P^T is in the registers exactly as the second product
// O^T = V^T P^T takes it (the sum over the keys runs in the order that the registers hold, V^T is read with the same order:
// ds_read_b64_tr_b16 for 16-bit types, four plain reads for float32).  The running maximum and sum are in 32 bits; P is rounded to
// the inputs' type for the second product, half a step of each weight; in float16 a weight keeps that down to 2^-25 of the row's largest (Range below).
// float32 runs on v_mfma_f32_16x16x4 (exact products), 16-bit types on v_mfma_f32_16x16x32.
// The backward recomputes P from lse; dq walks over keys, (dk, dv) over rows: no atomics, the same result every time.  P is rounded to the inputs' type for dv too; ds, which has both signs,
// goes into its products in two 16-bit pieces (rest_of below).  In float16 ds is taken times a power of two, of a row's own in dq and of a key's own in dk, and P times 2^14 in dv (Scaled below).
// Products run at a raised wave priority in the forward and dq: with two waves a SIMD one computes weights while the other holds the matrix pipe
// (forward 2 000 x 4 099, 64 heads of 128: 372 -> 360 us, dq of 1 500 x 2 049, 32 heads of 64: 69.4 -> 68.2; dk, dv: nothing).
// Bounds and figures (float16 / bfloat16 unless said): forward of 2 000 x 4 099, 64 heads of 128, 730 TFLOP/s, matrix pipe 30% and vector pipe 33% busy, the rest
// waits that two waves a SIMD (253 registers) do not hide.  One token on 48 x up to 8 192 states, 4 key heads of 128: 132 us, 4.6 TB/s where a large copy reaches 4.92, and 10 for the
// join of the splits: 145 a call.  float32 with heads of 16 (512 x 100 on 100): 66 us, bound by issue (products 33%, vector instructions 49%), half of the latter each wave's start and
// end.  Backward of 2 x 1 500 on up to 2 049, 16 / 4 heads of 64: dq 87 us, (dk, dv) 92 us (matrix pipe 20 and 24%, vector pipe 33 and 37% busy).
// Few rows: the key axis is split over workgroups and joined by a second launch.
// Non-finite values where nothing may look (a masked key whose value is NaN): 0 * NaN would spoil the products, so a workgroup
// whose accumulators end non-finite walks its tiles once more with the non-finite 16-byte pieces replaced by zeros and their
// contribution to the rows that do see them put back: a masked key never shows, a visible one does.
#include <type_traits>

#include "rr_types.h"

namespace {

#define RR_XA_KT 64            // keys (or rows) of a staged tile
#define RR_XA_PART(DP) ((DP) + 4)      // floats of a row's partial result: DP sums, the maximum, the sum of weights, two unused (16-byte pieces stay aligned)
#define RR_LOG2E 1.44269504088896340736f
#define RR_LN2 0.69314718055994530942f

struct XAttn {
  const void *q, *k, *v;
  void* out;
  float* lse;                            // [B][Hq][Lq] or NULL
  const uint8_t* mask;                   // [B][Hq][Lq][Lk] by strides, 1 = may be seen, or NULL
  const void* lens;                      // [B] int32 / int64 or NULL
  long long qb, ql, qh, kb, kl, kh, vb, vl, vh, mb, ml, mh;
  int lens64, B, Lq, Lk, Hk, G, D;
  float scale;
  int nsplit, tiles_per_split, nblk;     // splits of the walked axis, its tiles a split, workgroups along the kept axis
  int b0;                                // the launch's first batch entry
  float* part;                           // partial results of the splits
  // backward
  const void* dout;
  long long gb, gl, gh;
  float* delta;                          // [B][Hq][Lq]
  void *dq, *dk, *dv;                    // contiguous
};

template <typename T> struct Mx;
template <> struct Mx<float> {
  typedef f32x4 Frag;
  static constexpr int KC = 16, EPC = 4, PT = 1;          // contraction of a step, elements of 16 bytes, score tiles a second-product step takes
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag pack(const f32x4* p) { return p[0]; }
  static __device__ __forceinline__ Frag tr(const float* t, int pitch, int row0, int col0, int lane) {      // A = X^T: rows row0 + 4g + i, column col0 + lane % 16
    const float* p = t + (row0 + 4 * (lane >> 4)) * pitch + col0 + (lane & 15);
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = p[i * pitch];
    return f;
  }
};
typedef short rr_s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) rr_s16x4 rr_lds_s16x4;
template <typename T>
__device__ __forceinline__ void tr16(const T* t, int pitch, int row0, int col0, int lane, short (&f)[8]) {
  const int i = lane & 15;
  T* p = const_cast<T*>(t) + (row0 + 4 * (lane >> 4) + (i >> 2)) * pitch + col0 + 4 * (i & 3);
  const rr_s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rr_lds_s16x4*)p);
  const rr_s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((rr_lds_s16x4*)(p + 16 * pitch));
#pragma unroll
  for (int j = 0; j < 4; ++j) { f[j] = a[j]; f[4 + j] = b[j]; }
}
typedef short rr_s16x8 __attribute__((ext_vector_type(8)));
template <> struct Mx<rr_f16> {
  typedef rr_f16x8 Frag;
  static constexpr int KC = 32, EPC = 8, PT = 2;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ Frag pack(const f32x4* p) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = (rr_f16)p[0][i]; f[4 + i] = (rr_f16)p[1][i]; }
    return f;
  }
  static __device__ __forceinline__ Frag tr(const rr_f16* t, int pitch, int row0, int col0, int lane) {
    short f[8];
    tr16(t, pitch, row0, col0, lane, f);
    rr_s16x8 v = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
    return __builtin_bit_cast(Frag, v);
  }
};
template <> struct Mx<rr_bf16> {
  typedef rr_bf16x8 Frag;
  static constexpr int KC = 32, EPC = 8, PT = 2;
  static __device__ __forceinline__ f32x4 mma(Frag a, Frag b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static __device__ __forceinline__ Frag pack(const f32x4* p) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = (rr_bf16)p[0][i]; f[4 + i] = (rr_bf16)p[1][i]; }
    return f;
  }
  static __device__ __forceinline__ Frag tr(const rr_bf16* t, int pitch, int row0, int col0, int lane) {
    short f[8];
    tr16(t, pitch, row0, col0, lane, f);
    rr_s16x8 v = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7]};
    return __builtin_bit_cast(Frag, v);
  }
};

template <typename T> using FragOf = typename Mx<T>::Frag;
// What rounding to a 16-bit type took from two score tiles: the second piece of ds.  In one piece dq of narrow heads and of few queries was 1.5 to 1.7 times as far from 64 bits as its own
// rounding alone, dk 1.4 to 1.6; in two 1.0 to 1.3.  P, never negative, costs dv and the output a factor of 1.4 in one piece and keeps it.  Time of a second piece, bfloat16: 2 x 1 500 on
// 2 049, 16 / 4 heads of 64, every key seen, dq 69 -> 90 us, (dk, dv) 122 -> 139; one such of 128, 2 048 keys, 80 -> 93 and 119 -> 131; 64 x 101 on 103, 8 heads of 16, 9.1 -> 9.6 and 8.2 -> 8.8
template <typename T>
__device__ __forceinline__ FragOf<T> rest_of(const f32x4* x, const FragOf<T>& hi) {
  f32x4 r[2];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[0][i] = x[0][i] - (float)hi[i];
    r[1][i] = x[1][i] - (float)hi[4 + i];
  }
  return Mx<T>::pack(r);
}

template <typename T, int DP> struct Dims {
  static constexpr int KD = DP < Mx<T>::KC ? Mx<T>::KC : DP;      // columns of a staged row (zeros behind the head dim)
  static constexpr int NK = KD / Mx<T>::KC;                       // steps of the first product
  static constexpr int DT = DP / 16;                              // tiles of the second product
  // row pitches: 16 bytes more than the row lets 16 rows' 16-byte reads start in 16 different bank groups; transposed 16-bit
  // reads (four rows of 32 bytes a lane group) want 32
  static constexpr int PR = KD + 16 / (int)sizeof(T);
  static constexpr int PX = KD + (sizeof(T) == 2 ? 32 : 16) / (int)sizeof(T);
  static constexpr int CPR = KD / Mx<T>::EPC;                     // 16-byte pieces of a staged row
};

__device__ __forceinline__ bool nonfinite4(const float4& v, int is16) {
  const uint32_t w[4] = {__float_as_uint(v.x), __float_as_uint(v.y), __float_as_uint(v.z), __float_as_uint(v.w)};
  bool b = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (is16 == 0) b |= (w[i] & 0x7f800000u) == 0x7f800000u;
    else {
      const uint32_t e = is16 == 1 ? 0x7c00u : 0x7f80u;
      b |= (w[i] & e) == e || (w[i] >> 16 & e) == e;
    }
  }
  return b;
}
template <typename T> struct kind16;
template <> struct kind16<float> { static constexpr int v = 0; };
template <> struct kind16<rr_f16> { static constexpr int v = 1; };
template <> struct kind16<rr_bf16> { static constexpr int v = 2; };

// one row of the packed row list: group member r / Lq, position r % Lq
struct RowAt { int g, s; };
__device__ __forceinline__ RowAt row_at(int r, int Lq, int G) {
  if (G == 1) return {0, r};
  const int g = r / Lq;
  return {g, r - g * Lq};
}

// rows [row0, row0 + 64) of a tensor, 16-byte pieces over the 256 threads, on their way through registers into LDS (zeros behind the last row and the
// head dim): the loads of the next tile are in flight while the present one is computed
template <typename T, int DP>
struct Piece {
  using Dm = Dims<T, DP>;
  static constexpr int N = RR_XA_KT * Dm::CPR / 256;
  float4 v[N];
  // base: the tile's first row, ld: elements from row to row; rows: how many exist from there on.  A thread's pieces lie 256 / CPR rows apart.
  __device__ __forceinline__ void load(const T* base, long long ld, int rows, int D) {
    const int row = threadIdx.x / Dm::CPR, col = threadIdx.x % Dm::CPR * Mx<T>::EPC;
    const long long off = row * ld + col;
    if (rows >= RR_XA_KT && D == Dm::KD) {                               // (uniform: a whole tile needs no conditions)
#pragma unroll
      for (int c = 0; c < N; ++c) v[c] = *reinterpret_cast<const float4*>(base + c * (256 / Dm::CPR) * ld + off);
    } else {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row + c * (256 / Dm::CPR) < rows && col < D) v[c] = *reinterpret_cast<const float4*>(base + c * (256 / Dm::CPR) * ld + off);
      }
    }
  }
  // safe: pieces that hold a non-finite value become zeros and their row's bit is set in `flag`
  template <int PITCH>
  __device__ __forceinline__ void store(T* lds, bool safe, uint32_t* flag) {
#pragma unroll
    for (int c = 0; c < N; ++c) {
      const int i = threadIdx.x + 256 * c, row = i / Dm::CPR, ch = i % Dm::CPR;
      if (safe && nonfinite4(v[c], kind16<T>::v)) {
        v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
        atomicOr(&flag[row >> 5], 1u << (row & 31));
      }
      *reinterpret_cast<float4*>(lds + row * PITCH + ch * Mx<T>::EPC) = v[c];
    }
  }
};
__device__ __forceinline__ void clear_flag(uint32_t* flag) {             // (by the whole workgroup)
  if (threadIdx.x < 2) flag[threadIdx.x] = 0u;
  __syncthreads();
}

template <typename T>
__device__ __forceinline__ FragOf<T> frag_at(const T* p) { return *reinterpret_cast<const FragOf<T>*>(p); }
template <typename T>
__device__ __forceinline__ FragOf<T> frag_zero() {
  FragOf<T> f;
#pragma unroll
  for (int i = 0; i < Mx<T>::EPC; ++i) f[i] = (T)0.f;
  return f;
}

__device__ __forceinline__ int seen_keys(const XAttn& a, int b) {
  if (a.lens == nullptr) return a.Lk;
  const long long n = a.lens64 ? ((const long long*)a.lens)[b] : (long long)((const int*)a.lens)[b];
  return n < 0 ? 0 : n > a.Lk ? a.Lk : (int)n;
}
// four consecutive mask bytes of a row from `key` on, zeros behind the end: one unaligned 4-byte load that ends inside the row
__device__ __forceinline__ uint32_t mask4(const uint8_t* row, int key, int Lk) {
  uint32_t m = 0;
  if (Lk >= 4) {                                                         // (uniform)
    const int from = key < Lk - 4 ? key : Lk - 4, off = key - from;
    __builtin_memcpy(&m, row + from, 4);
    return off < 4 ? m >> (8 * off) : 0u;
  }
  for (int i = 0; i < Lk; ++i) m |= (uint32_t)row[i] << (8 * i);
  return key < 4 ? m >> (8 * key) : 0u;
}
// the same at key k0 + i of a tile; whole tiles need none of the conditions (WHOLE: where there are registers for both)
template <bool WHOLE>
__device__ __forceinline__ uint32_t mask_at(const uint8_t* row, int k0, int i, int Lk) {
  uint32_t m;
  if (WHOLE && k0 + RR_XA_KT <= Lk) __builtin_memcpy(&m, row + k0 + i, 4);          // (uniform)
  else m = mask4(row, k0 + i, Lk);
  return m;
}
__device__ __forceinline__ uint32_t first_bytes(uint32_t b, int n) {     // the first n of four bytes
  return n >= 4 ? b : n <= 0 ? 0u : b & ((1u << (8 * n)) - 1u);
}
// x where the byte of its place is 1, y where it is 0.  By bit fields (two instructions a value, three with comparisons) and without branches: the four values stay
// in their registers
__device__ __forceinline__ void keep4(f32x4& x, uint32_t bytes, float y) {
  f32x4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t k = (uint32_t)__builtin_amdgcn_sbfe((int)bytes, 8 * i, 1);
    r[i] = __uint_as_float((__float_as_uint(x[i]) & k) | (__float_as_uint(y) & ~k));
  }
  x = r;
}
// the flags of four consecutive rows of a tile as bytes
__device__ __forceinline__ uint32_t flag4(const uint32_t* flag, int row) {
  const uint32_t f = flag[row >> 5] >> (row & 31);
  return (f & 1u) | (f & 2u) << 7 | (f & 4u) << 14 | (f & 8u) << 21;
}
__device__ __forceinline__ float group_max(float v) { v = fmaxf(v, __shfl_xor(v, 16)); return fmaxf(v, __shfl_xor(v, 32)); }
__device__ __forceinline__ float group_sum(float v) { v += __shfl_xor(v, 16); return v + __shfl_xor(v, 32); }
__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.f : m; }
// a row's log-sum-exp in powers of two; +inf where it has no weight at all: all its weights are then exp2(score - inf) = 0
__device__ __forceinline__ float lse2_of(float lse) { return lse == -INFINITY ? INFINITY : lse * RR_LOG2E; }
__device__ __forceinline__ bool is_bad(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

// the wave's QT x 16 rows as B operands (lane: row lane % 16, 16 bytes at piece lane / 16 of every contraction step)
template <typename T, int DP, int QT, typename F>
__device__ __forceinline__ void load_rows(F& f, const T* base, long long sl, long long sh, int row0, int R, const XAttn& a, int lane) {
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + (lane & 15);
    const RowAt at = row_at(r < R ? r : R - 1, a.Lq, a.G);
    const T* p = base + at.s * sl + at.g * sh;
#pragma unroll
    for (int k = 0; k < Dims<T, DP>::NK; ++k) {
      const int c = k * Mx<T>::KC + (lane >> 4) * Mx<T>::EPC;
      f[t][k] = r < R && c < a.D ? frag_at<T>(p + c) : frag_zero<T>();
    }
  }
}

struct Blk { int b, hk, split, blk; };
__device__ __forceinline__ Blk block_of(const XAttn& a) {
  // workgroups go to the eight XCDs in turn: each gets one stretch of the work, so that the heads of an instance, which share its cache lines and
  // its mask, meet in one L2
  const unsigned n = gridDim.x, x = blockIdx.x & 7u, q = n >> 3, r = n & 7u;
  unsigned i = x * q + (x < r ? x : r) + (blockIdx.x >> 3);
  Blk w;
  w.blk = (int)(i % (unsigned)a.nblk); i /= (unsigned)a.nblk;
  w.split = (int)(i % (unsigned)a.nsplit); i /= (unsigned)a.nsplit;
  w.hk = (int)(i % (unsigned)a.Hk);
  w.b = a.b0 + (int)(i / (unsigned)a.Hk);
  return w;
}

// ------------------------------------------------------------------------------------------------ forward
// registers: two waves a SIMD, except where 128-wide float32 rows need more
// Variants near the register limit keep the reads of one 16-key step behind those of the step before (hoisted further, they spill)
template <bool TIGHT>
__device__ __forceinline__ void in_order() {
  if constexpr (TIGHT) __builtin_amdgcn_sched_barrier(0);
}
// A row's weights are taken relative to 2^(its running maximum - UP), and the running maximum moves only when a score passes it by 2^SLACK: weights up to that are as exact as those up
// to one, and a tile that does not move it needs no exchange between the lanes of a row and no rescaling.  float16 has 2^15 above one and 2^-14 below: with UP
// the largest weight stands between 2^11 and 2^15 instead of 1 and 2^8, so that small ones keep their bits (20 000 keys of 1.47 2^-24 beside one of 1 lost a third of their sum)
template <typename T> struct Range { static constexpr float UP = 0.f, SLACK = 8.f; };
template <> struct Range<rr_f16> { static constexpr float UP = 11.f, SLACK = 4.f; };
// float16 in the backward.  ds = p (do.v - delta) may be of any size: a mean loss over long states leaves 1e-7 and less, large gradients on few keys pass 65 504 though dq and dk fit.  The
// second products take ds 2^n, n of a row's (a key's) own, undone in 32 bits at the end.  n begins at 60 and falls, the sums with it, whenever a value would pass 2^15: to where the largest
// of the step stands at 2^9 .. 2^10, so that it rarely falls again.  Then the rounding of a small ds is off by 2^-34 of the row's (key's) largest at the most.  P <= 1 is taken times
// 2^14: off by 2^-39 at the most.  It costs a comparison and a branch for
// every 32 keys (rows) of a row (key) and dk a product for each weight; bfloat16, which has float32's exponents, does without.  float16 against bfloat16: 2 x 1 500 on 2 049, 16 / 4 heads of
// 64, every key seen, dq 96 and 89 us, (dk, dv) 158 and 139; 120 on 60, 2 048 heads of 64, 58 and 53, 40 and 37
#define RR_XA_UP 0x1p60f
#define RR_XA_P_BITS 14
template <typename T> struct Scaled { static constexpr bool v = std::is_same_v<T, rr_f16>; };
__device__ __forceinline__ float abs4(float mx, const f32x4& x) { return fmaxf(fmaxf(fmaxf(fabsf(x[0]), fabsf(x[1])), fmaxf(fabsf(x[2]), fabsf(x[3]))), mx); }
// the power of two that a largest value of `mx` asks for, 1 where it needs none (or is not finite: the sums are then, too)
__device__ __forceinline__ float fall_by(float mx) { return mx > 32768.f && mx < INFINITY ? ldexpf(1.f, 10 - __builtin_amdgcn_frexp_expf(mx)) : 1.f; }
template <typename T, int DP> struct Waves { static constexpr int N = sizeof(T) == 4 && DP == 128 ? 1 : 2; };

template <typename T, int DP, int QT>
__global__ __launch_bounds__(256, (Waves<T, DP>::N)) void k_xattn_fwd(XAttn a) {
  using M = Mx<T>;
  using Dm = Dims<T, DP>;
  constexpr bool TIGHT = DP == 128 && QT == 2, SKIP = sizeof(T) == 4;
  __shared__ __attribute__((aligned(16))) T sk[2][RR_XA_KT * Dm::PR];
  __shared__ __attribute__((aligned(16))) T sv[2][RR_XA_KT * Dm::PX];
  __shared__ uint32_t flag[2][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const Blk w = block_of(a);
  const int R = a.G * a.Lq, row0 = (w.blk * 4 + wave) * 16 * QT;
  const bool busy = row0 < R;
  const int seen = seen_keys(a, w.b);
  const T* kp = (const T*)a.k + (long long)w.b * a.kb + (long long)w.hk * a.kh;
  const T* vp = (const T*)a.v + (long long)w.b * a.vb + (long long)w.hk * a.vh;
  auto krow = [&](int r) { return kp + (long long)r * a.kl; };
  auto vrow = [&](int r) { return vp + (long long)r * a.vl; };
  const int first = w.split * a.tiles_per_split * RR_XA_KT;
  int last = first + a.tiles_per_split * RR_XA_KT;
  last = last < seen ? last : seen;
  Piece<T, DP> pk, pv;
  if (first < last) {
    pk.load(krow(first), a.kl, seen - first, a.D);
    pv.load(vrow(first), a.vl, seen - first, a.D);
  }
  typename M::Frag qf[QT][Dm::NK];
  load_rows<T, DP, QT>(qf, (const T*)a.q + (long long)w.b * a.qb + (long long)w.hk * a.G * a.qh, a.ql, a.qh, row0, R, a, lane);
  const uint8_t* mrow[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + j;
    const RowAt at = row_at(r < R ? r : R - 1, a.Lq, a.G);
    mrow[t] = a.mask + w.b * a.mb + (w.hk * a.G + at.g) * a.mh + at.s * a.ml;
  }
  const float c2 = a.scale * RR_LOG2E;
  f32x4 o[QT][Dm::DT];
  float m[QT], l[QT];
  // one staged tile; `safe`: second walk.  float32 skips 16-key tiles behind the last key; 16-bit types compute them and drop the scores: branches between the
  // tiles keep the reads of the next one from being issued early, which costs more than the products
  auto tile = [&](auto safe, int k0, int at) {
    const T *tk = sk[at], *tv = sv[at];
    uint32_t mb[QT][4];
    if (a.mask != nullptr) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int n = 0; n < 4; ++n) mb[t][n] = mask_at<!TIGHT>(mrow[t], k0, 16 * n + 4 * g, a.Lk);
    }
    __builtin_amdgcn_s_setprio(1);
    const int parts = SKIP ? (seen - k0 + 15) >> 4 : 4;
    f32x4 s[QT][4];
#pragma unroll
    for (int n = 0; n < 4; ++n) {
#pragma unroll
      for (int t = 0; t < QT; ++t) s[t][n] = rr_zero4();
      if (!SKIP || n < parts) {
#pragma unroll
        for (int k = 0; k < Dm::NK; ++k) {
          const typename M::Frag f = frag_at<T>(tk + (16 * n + j) * Dm::PR + k * M::KC + g * M::EPC);
#pragma unroll
          for (int t = 0; t < QT; ++t) s[t][n] = M::mma(f, qf[t][k], s[t][n]);
        }
      }
      in_order<TIGHT>();
    }
    __builtin_amdgcn_s_setprio(0);
    if (a.mask != nullptr || k0 + RR_XA_KT > seen) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          if (SKIP && n >= parts) continue;
          uint32_t b = a.mask != nullptr ? mb[t][n] : 0x01010101u;
          if (k0 + RR_XA_KT > seen) b = first_bytes(b, seen - (k0 + 16 * n + 4 * g));
          keep4(s[t][n], b, -INFINITY);
        }
    }
    float mx[QT];
    bool move = false;
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      mx[t] = s[t][0][0];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (SKIP && n >= parts) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) mx[t] = fmaxf(mx[t], s[t][n][i]);
      }
      move |= mx[t] * c2 > m[t] + (Range<T>::UP + Range<T>::SLACK);
    }
    if (__any(move)) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float mn = fmaxf(m[t], group_max(mx[t]) * c2 - Range<T>::UP);
        const float al = __builtin_amdgcn_exp2f(m[t] - finite_or_zero(mn));
        l[t] *= al;
        m[t] = mn;
#pragma unroll
        for (int d = 0; d < Dm::DT; ++d) o[t][d] *= al;
      }
    }
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      const float mu = finite_or_zero(m[t]);
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (SKIP && n >= parts) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[t][n][i] = __builtin_amdgcn_exp2f(fmaf(s[t][n][i], c2, -mu));
          sum += s[t][n][i];
        }
      }
      l[t] += sum;
    }
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int n = 0; n < 4; n += M::PT) {
      if (SKIP && n >= parts) break;
      typename M::Frag pf[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) pf[t] = M::pack(&s[t][n]);
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) {
        const typename M::Frag f = M::tr(tv, Dm::PX, 16 * n, 16 * d, lane);
#pragma unroll
        for (int t = 0; t < QT; ++t) o[t][d] = M::mma(f, pf[t], o[t][d]);
        if ((d & 3) == 3) in_order<TIGHT>();
      }
    }
    __builtin_amdgcn_s_setprio(0);
    const uint32_t* fl = flag[at];
    if constexpr (safe()) if (fl[0] | fl[1]) {               // rare: what visible keys hold in the pieces that were zeroed
#pragma unroll
      for (int n = 0; n < 4; ++n)
        for (int kk = 0; kk < 16; ++kk) {
          const int key = 16 * n + kk;
          if (!(fl[key >> 5] >> (key & 31) & 1u)) continue;
          const T* vr = vrow(k0 + key);
#pragma unroll
          for (int t = 0; t < QT; ++t) {
            const float mine = (kk & 3) == 0 ? s[t][n][0] : (kk & 3) == 1 ? s[t][n][1] : (kk & 3) == 2 ? s[t][n][2] : s[t][n][3];
            const float p = __shfl(mine, j + 16 * (kk >> 2));
#pragma unroll
            for (int d = 0; d < Dm::DT; ++d) {
              const int c = 16 * d + 4 * g, piece = c / M::EPC * M::EPC;
              if (p == 0.f || c >= a.D || !nonfinite4(*reinterpret_cast<const float4*>(vr + piece), kind16<T>::v)) continue;
#pragma unroll
              for (int i = 0; i < 4; ++i) o[t][d][i] += p * (float)vr[c + i];
            }
          }
        }
    }
  };
  auto walk = [&](auto safe) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      m[t] = -INFINITY; l[t] = 0.f;
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) o[t][d] = rr_zero4();
    }
    if constexpr (safe()) {
      clear_flag(flag[0]);
      pk.load(krow(first), a.kl, seen - first, a.D);
      pv.load(vrow(first), a.vl, seen - first, a.D);
    }
    if (first < last) {
      pk.template store<Dm::PR>(sk[0], false, flag[0]);
      pv.template store<Dm::PX>(sv[0], safe(), flag[0]);
    }
    __syncthreads();
    int at = 0;
    for (int k0 = first; k0 < last; k0 += RR_XA_KT, at ^= 1) {
      const bool more = k0 + RR_XA_KT < last;
      if (more) {
        pk.load(krow(k0 + RR_XA_KT), a.kl, seen - k0 - RR_XA_KT, a.D);
        pv.load(vrow(k0 + RR_XA_KT), a.vl, seen - k0 - RR_XA_KT, a.D);
      }
      if (busy) tile(safe, k0, at);
      if (more) {
        if constexpr (safe()) clear_flag(flag[at ^ 1]);
        pk.template store<Dm::PR>(sk[at ^ 1], false, flag[at ^ 1]);
        pv.template store<Dm::PX>(sv[at ^ 1], safe(), flag[at ^ 1]);
      }
      __syncthreads();
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= is_bad(o[t][d][i]);
    return __syncthreads_or(bad && busy);
  };
  if (walk(std::false_type{})) walk(std::true_type{});
  if (!busy) return;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + j;
    const float lt = group_sum(l[t]);
    if (r >= R) continue;
    const RowAt at = row_at(r, a.Lq, a.G);
    const int head = w.hk * a.G + at.g;
    if (a.nsplit > 1) {                            // partials: [B * Hk * R][nsplit][RR_XA_PART] floats
      float* p = a.part + (((long long)(w.b * a.Hk + w.hk) * R + r) * a.nsplit + w.split) * RR_XA_PART(DP);
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) *reinterpret_cast<f32x4*>(p + 16 * d + 4 * g) = o[t][d];
      if (g == 0) { p[DP] = m[t]; p[DP + 1] = lt; }
    } else {
      const float inv = lt == 0.f ? 0.f : 1.0f / lt;
      T* dst = (T*)a.out + (((long long)w.b * a.Lq + at.s) * (a.Hk * a.G) + head) * a.D;
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) {
        const int c = 16 * d + 4 * g;
        if (c < a.D) {
          typedef T V4 __attribute__((ext_vector_type(4)));
          V4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = (T)(o[t][d][i] * inv);
          *reinterpret_cast<V4*>(dst + c) = v;
        }
      }
      if (a.lse != nullptr && g == 0)
        a.lse[((long long)w.b * (a.Hk * a.G) + head) * a.Lq + at.s] = lt == 0.f ? -INFINITY : (m[t] + __log2f(lt)) * RR_LN2;
    }
  }
}

// joins the splits of a row: DP / 4 lanes a row, four columns each
template <typename T, int DP>
__global__ __launch_bounds__(256) void k_xattn_join(XAttn a) {
  constexpr int LPR = DP / 4;
  const int c = threadIdx.x % LPR * 4;
  const long long row = (long long)blockIdx.x * (256 / LPR) + threadIdx.x / LPR;
  const int R = a.G * a.Lq;
  if (row >= (long long)a.B * a.Hk * R) return;
  const float* p = a.part + row * a.nsplit * RR_XA_PART(DP);
  float m = -INFINITY;
  for (int i = 0; i < a.nsplit; ++i) m = fmaxf(m, p[i * RR_XA_PART(DP) + DP]);
  const float mu = finite_or_zero(m);
  f32x4 acc = rr_zero4();
  float l = 0.f;
#pragma unroll 4
  for (int i = 0; i < a.nsplit; ++i) {
    const float* pi = p + i * RR_XA_PART(DP);
    const float mi = pi[DP], li = pi[DP + 1], f = __builtin_amdgcn_exp2f(mi - mu);
    const f32x4 v = *reinterpret_cast<const f32x4*>(pi + c);
    l = fmaf(li, f, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] = mi == -INFINITY ? acc[e] : fmaf(v[e], f, acc[e]);
  }
  const int b = (int)(row / ((long long)a.Hk * R)), hk = (int)(row / R % a.Hk);
  const RowAt at = row_at((int)(row % R), a.Lq, a.G);
  const int head = hk * a.G + at.g;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  T* dst = (T*)a.out + (((long long)b * a.Lq + at.s) * (a.Hk * a.G) + head) * a.D;
  if (c < a.D) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    const V4 v = {(T)(acc[0] * inv), (T)(acc[1] * inv), (T)(acc[2] * inv), (T)(acc[3] * inv)};
    *reinterpret_cast<V4*>(dst + c) = v;
  }
  if (a.lse != nullptr && c == 0) a.lse[((long long)b * (a.Hk * a.G) + head) * a.Lq + at.s] = l == 0.f ? -INFINITY : (m + __log2f(l)) * RR_LN2;
}

// ------------------------------------------------------------------------------------------------ backward: dq (walks over the keys)
// ONE: all keys lie in one tile.  delta is then sum p (do.v) over it instead of do.out, whose stored out is rounded to 16 bits: with few keys that rounding is as
// large as the differences do.v - delta (2 keys: dq and dk off by 2.2 times what their own rounding costs, 1.4 with the sum over the tile).  The first walk takes it and the second keeps
// it: there the pieces of a visible key that hold a non-finite value are zeros, and the key's score would be another
template <typename T, int DP, int QT, bool ONE>
__global__ __launch_bounds__(256, (Waves<T, DP>::N)) void k_xattn_dq(XAttn a) {
  using M = Mx<T>;
  using Dm = Dims<T, DP>;
  constexpr bool TIGHT = DP == 128 && QT == 2, SKIP = sizeof(T) == 4;
  static constexpr int STEPS = sizeof(T) == 2 && (ONE || DP == 128) ? 1 : 4;      // of a tile, unrolled (those spill if they are; the others gain 4%)
  __shared__ __attribute__((aligned(16))) T sk[2][RR_XA_KT * Dm::PX];
  __shared__ __attribute__((aligned(16))) T sv[2][RR_XA_KT * Dm::PR];
  __shared__ uint32_t flag[2][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const Blk w = block_of(a);
  const int R = a.G * a.Lq, H = a.G * a.Hk, row0 = (w.blk * 4 + wave) * 16 * QT;
  const bool busy = row0 < R;
  const int seen = seen_keys(a, w.b);
  const T* kp = (const T*)a.k + (long long)w.b * a.kb + (long long)w.hk * a.kh;
  const T* vp = (const T*)a.v + (long long)w.b * a.vb + (long long)w.hk * a.vh;
  auto krow = [&](int r) { return kp + (long long)r * a.kl; };
  auto vrow = [&](int r) { return vp + (long long)r * a.vl; };
  const int first = w.split * a.tiles_per_split * RR_XA_KT;
  int last = first + a.tiles_per_split * RR_XA_KT;
  last = last < seen ? last : seen;
  Piece<T, DP> pk, pv;
  if (first < last) {
    pk.load(krow(first), a.kl, seen - first, a.D);
    pv.load(vrow(first), a.vl, seen - first, a.D);
  }
  typename M::Frag qf[QT][Dm::NK], gf[QT][Dm::NK];
  load_rows<T, DP, QT>(qf, (const T*)a.q + (long long)w.b * a.qb + (long long)w.hk * a.G * a.qh, a.ql, a.qh, row0, R, a, lane);
  load_rows<T, DP, QT>(gf, (const T*)a.dout + (long long)w.b * a.gb + (long long)w.hk * a.G * a.gh, a.gl, a.gh, row0, R, a, lane);
  const uint8_t* mrow[QT];
  float lse2[QT], delta[QT];
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + j, rc = r < R ? r : R - 1;
    const RowAt at = row_at(rc, a.Lq, a.G);
    const int head = w.hk * a.G + at.g;
    mrow[t] = a.mask + w.b * a.mb + head * a.mh + at.s * a.ml;
    const long long li = ((long long)w.b * H + head) * a.Lq + at.s;
    lse2[t] = busy && r < R ? lse2_of(a.lse[li]) : 0.f;
    const T* op = (const T*)a.out + (((long long)w.b * a.Lq + at.s) * H + head) * a.D;
    float d = 0.f;
#pragma unroll
    for (int k = 0; k < Dm::NK; ++k) {
      const int c = k * M::KC + g * M::EPC;
      if (r < R && c < a.D) {
        const typename M::Frag of = frag_at<T>(op + c);
#pragma unroll
        for (int i = 0; i < M::EPC; ++i) d = fmaf((float)of[i], (float)gf[t][k][i], d);
      }
    }
    delta[t] = group_sum(d);
    if (!ONE && w.split == 0 && g == 0 && r < R) a.delta[li] = delta[t];
  }
  const float c2 = a.scale * RR_LOG2E;
  f32x4 o[QT][Dm::DT];
  float up[QT];
  // keys behind the last one are staged as zeros: whatever their weight, they add nothing (unless it overflows, which the second walk sorts out)
  auto tile = [&](auto safe, int k0, int at) {
    const T *tk = sk[at], *tv = sv[at];
    const uint32_t* fl = flag[at];
    const bool some = a.mask != nullptr || safe() || (Scaled<T>::v && k0 + RR_XA_KT > seen);      // (uniform) not every pair of the tile may be seen
    uint32_t mb[QT][4];
    if (a.mask != nullptr) {
#pragma unroll
      for (int t = 0; t < QT; ++t)
#pragma unroll
        for (int n = 0; n < 4; ++n) mb[t][n] = mask_at<!TIGHT>(mrow[t], k0, 16 * n + 4 * g, a.Lk);
    }
    float dsum[QT];
#pragma unroll
    for (int t = 0; t < QT; ++t) dsum[t] = 0.f;
#pragma unroll 1
    for (int phase = ONE && !safe() ? 0 : 1; phase < 2; ++phase) {
    if (ONE && !safe()) asm volatile("" ::: "memory");       // or the compiler lifts the tile's reads out of the loop over the phases, and keeps them in scratch memory
#pragma unroll STEPS
    for (int n = 0; n < 4; n += M::PT) {
      if (SKIP && k0 + 16 * n >= seen) break;
      f32x4 s[QT][M::PT], dp[QT][M::PT];
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int u = 0; u < M::PT; ++u) {
#pragma unroll
        for (int t = 0; t < QT; ++t) { s[t][u] = rr_zero4(); dp[t][u] = rr_zero4(); }
#pragma unroll
        for (int k = 0; k < Dm::NK; ++k) {
          const typename M::Frag fk = frag_at<T>(tk + (16 * (n + u) + j) * Dm::PX + k * M::KC + g * M::EPC);
          const typename M::Frag fv = frag_at<T>(tv + (16 * (n + u) + j) * Dm::PR + k * M::KC + g * M::EPC);
#pragma unroll
          for (int t = 0; t < QT; ++t) { s[t][u] = M::mma(fk, qf[t][k], s[t][u]); dp[t][u] = M::mma(fv, gf[t][k], dp[t][u]); }
        }
        in_order<TIGHT>();
      }
      __builtin_amdgcn_s_setprio(0);
      if (ONE && !safe() && phase == 0) {
#pragma unroll
        for (int t = 0; t < QT; ++t)
#pragma unroll
          for (int u = 0; u < M::PT; ++u) {
            f32x4 x;
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_exp2f(fmaf(s[t][u][i], c2, -lse2[t])) * dp[t][u][i];
            keep4(x, first_bytes(a.mask != nullptr ? mb[t][n + u] : 0x01010101u, seen - (k0 + 16 * (n + u) + 4 * g)), 0.f);
            dsum[t] += (x[0] + x[1]) + (x[2] + x[3]);
          }
        continue;
      }
      typename M::Frag pf[QT], pr[QT];
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const float ud = Scaled<T>::v ? delta[t] * up[t] : delta[t];
#pragma unroll
        for (int u = 0; u < M::PT; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[t][u][i], c2, -lse2[t]));
            s[t][u][i] = p * (Scaled<T>::v ? fmaf(dp[t][u][i], up[t], -ud) : dp[t][u][i] - ud);
          }
        if (some) {
#pragma unroll
          for (int u = 0; u < M::PT; ++u) {
            const int key = 16 * (n + u) + 4 * g;
            if constexpr (safe()) keep4(s[t][u], ~(flag4(fl, key) * 0xffu), __builtin_nanf(""));      // a visible key that holds a non-finite value
            keep4(s[t][u], first_bytes(a.mask != nullptr ? mb[t][n + u] : 0x01010101u, seen - (k0 + key)), 0.f);
          }
        }
        if constexpr (Scaled<T>::v) {
          const float mx = abs4(abs4(0.f, s[t][0]), s[t][M::PT - 1]);
          if (__any(mx > 32768.f)) {
            const float r = fall_by(group_max(mx));
            up[t] *= r;
#pragma unroll
            for (int u = 0; u < M::PT; ++u) s[t][u] *= r;
#pragma unroll
            for (int d = 0; d < Dm::DT; ++d) o[t][d] *= r;
          }
        }
        pf[t] = M::pack(s[t]);
        if constexpr (sizeof(T) == 2) pr[t] = rest_of<T>(s[t], pf[t]);
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) {
        const typename M::Frag f = M::tr(tk, Dm::PX, 16 * n, 16 * d, lane);
#pragma unroll
        for (int t = 0; t < QT; ++t) {
          o[t][d] = M::mma(f, pf[t], o[t][d]);
          if constexpr (sizeof(T) == 2) o[t][d] = M::mma(f, pr[t], o[t][d]);
        }
        if ((d & 3) == 3) in_order<TIGHT>();
      }
      __builtin_amdgcn_s_setprio(0);
    }
    if (ONE && !safe() && phase == 0) {
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        delta[t] = group_sum(dsum[t]);
        const int r = row0 + 16 * t + j;
        if (g == 0 && r < R) {
          const RowAt at = row_at(r, a.Lq, a.G);
          a.delta[((long long)w.b * H + w.hk * a.G + at.g) * a.Lq + at.s] = delta[t];
        }
      }
    }
    }
  };
  auto walk = [&](auto safe) {
#pragma unroll
    for (int t = 0; t < QT; ++t) {
      up[t] = RR_XA_UP;
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) o[t][d] = rr_zero4();
    }
    if constexpr (safe()) {
      clear_flag(flag[0]);
      pk.load(krow(first), a.kl, seen - first, a.D);
      pv.load(vrow(first), a.vl, seen - first, a.D);
    }
    if (first < last) {
      pk.template store<Dm::PX>(sk[0], safe(), flag[0]);
      pv.template store<Dm::PR>(sv[0], false, flag[0]);
    }
    __syncthreads();
    int at = 0;
    for (int k0 = first; k0 < last; k0 += RR_XA_KT, at ^= 1) {
      const bool more = !ONE && k0 + RR_XA_KT < last;
      if (more) {
        pk.load(krow(k0 + RR_XA_KT), a.kl, seen - k0 - RR_XA_KT, a.D);
        pv.load(vrow(k0 + RR_XA_KT), a.vl, seen - k0 - RR_XA_KT, a.D);
      }
      if (busy) tile(safe, k0, at);
      if (more) {
        if constexpr (safe()) clear_flag(flag[at ^ 1]);
        pk.template store<Dm::PX>(sk[at ^ 1], safe(), flag[at ^ 1]);
        pv.template store<Dm::PR>(sv[at ^ 1], false, flag[at ^ 1]);
      }
      __syncthreads();
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < QT; ++t)
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= is_bad(o[t][d][i]);
    return __syncthreads_or(bad && busy);
  };
  if constexpr (ONE)
    if (first >= last && busy)                                             // no key at all: nothing reads a weight, but delta is read
#pragma unroll
      for (int t = 0; t < QT; ++t) {
        const int r = row0 + 16 * t + j;
        const RowAt at = row_at(r < R ? r : R - 1, a.Lq, a.G);
        if (g == 0 && r < R) a.delta[((long long)w.b * H + w.hk * a.G + at.g) * a.Lq + at.s] = 0.f;
      }
  if (walk(std::false_type{})) walk(std::true_type{});
  if (!busy) return;
#pragma unroll
  for (int t = 0; t < QT; ++t) {
    const int r = row0 + 16 * t + j;
    if (r >= R) continue;
    const RowAt at = row_at(r, a.Lq, a.G);
    const long long at_out = (((long long)w.b * a.Lq + at.s) * H + w.hk * a.G + at.g) * a.D;
    float* p = a.part + (long long)w.split * a.B * a.Lq * H * a.D + at_out;
#pragma unroll
    for (int d = 0; d < Dm::DT; ++d) {
      const int c = 16 * d + 4 * g;
      if (c >= a.D) continue;
      const f32x4 x = (Scaled<T>::v ? o[t][d] * (1.f / up[t]) : o[t][d]) * a.scale;
      if (a.nsplit > 1) {
        *reinterpret_cast<f32x4*>(p + c) = x;
      } else {
        typedef T V4 __attribute__((ext_vector_type(4)));
        V4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = (T)x[i];
        *reinterpret_cast<V4*>((T*)a.dq + at_out + c) = v;
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ backward: dk, dv (walks over the rows)
template <typename T, int DP, int KW>        // KW x 16 keys a wave
__global__ __launch_bounds__(256, (DP == 128 ? 1 : 2)) void k_xattn_dkv(XAttn a) {
  using M = Mx<T>;
  using Dm = Dims<T, DP>;
  constexpr bool TIGHT = DP >= 64 && KW == 2, SKIP = sizeof(T) == 4;
  // steps of a tile, unrolled.  128 columns spill if they are: 16 query heads of 1 500, 4 of 2 048 keys took 264 us, 218 as a loop
  static constexpr int STEPS = sizeof(T) == 2 && DP >= 64 ? 1 : 4;
  constexpr int MP = RR_XA_KT + 4;           // a key's mask bytes of the tile's rows: a lane reads those of its four rows at once
  __shared__ __attribute__((aligned(16))) T sq[2][RR_XA_KT * Dm::PX];
  __shared__ __attribute__((aligned(16))) T sg[2][RR_XA_KT * Dm::PX];
  __shared__ __attribute__((aligned(16))) float sl[2][RR_XA_KT], sd[2][RR_XA_KT];
  __shared__ __attribute__((aligned(16))) uint8_t sm[2][64 * KW * MP];
  __shared__ uint32_t flag[2][2];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, j = lane & 15, g = lane >> 4;
  const Blk w = block_of(a);
  const int H = a.G * a.Hk, per_head = (a.Lq + RR_XA_KT - 1) / RR_XA_KT, block0 = w.blk * 64 * KW, key0 = block0 + wave * 16 * KW;
  const int seen = seen_keys(a, w.b);
  const bool busy = key0 < seen;
  const T* kp = (const T*)a.k + (long long)w.b * a.kb + (long long)w.hk * a.kh;
  const T* vp = (const T*)a.v + (long long)w.b * a.vb + (long long)w.hk * a.vh;
  const T* qp = (const T*)a.q + (long long)w.b * a.qb + (long long)w.hk * a.G * a.qh;
  const T* gp = (const T*)a.dout + (long long)w.b * a.gb + (long long)w.hk * a.G * a.gh;
  const float c2 = a.scale * RR_LOG2E;
  // the walked tiles: 64 positions of one head of the group each, head after head
  const int first = w.split * a.tiles_per_split;
  int last = first + a.tiles_per_split;
  last = block0 < seen ? (last < a.G * per_head ? last : a.G * per_head) : first;      // (a workgroup behind the last key only writes zeros)
  Piece<T, DP> pq, pg;
  float nl = 0.f, nd = 0.f;                                              // the tile's lse (in powers of two) and delta, a row a thread
  uint32_t nm[4 * KW];                                                   // its mask: KW times four keys' bytes of four rows a thread
  const int mrow = threadIdx.x / (16 * KW) * 4;                          // the first of them
  auto load_tile = [&](int tile) {
    const int h = tile / per_head, s0 = (tile - h * per_head) * RR_XA_KT, rows = a.Lq - s0, head = w.hk * a.G + h;
    pq.load(qp + h * a.qh + s0 * a.ql, a.ql, rows, a.D);
    pg.load(gp + h * a.gh + s0 * a.gl, a.gl, rows, a.D);
    if (threadIdx.x < RR_XA_KT) {
      const long long li = ((long long)w.b * H + head) * a.Lq + s0 + ((int)threadIdx.x < rows ? (int)threadIdx.x : rows - 1);
      nl = (int)threadIdx.x < rows ? lse2_of(a.lse[li]) - (Scaled<T>::v ? RR_XA_P_BITS : 0) : INFINITY;
      nd = (int)threadIdx.x < rows ? a.delta[li] : 0.f;
    }
    if (a.mask != nullptr) {
      const uint8_t* mp = a.mask + w.b * a.mb + head * a.mh + s0 * a.ml;
      const int key = block0 + threadIdx.x % (16 * KW) * 4;
#pragma unroll
      for (int c = 0; c < 4 * KW; ++c) {
        const int r = mrow + c / 4 * (256 / (4 * KW)) + c % 4;
        nm[c] = mask4(mp + (r < rows ? r : rows - 1) * a.ml, key, a.Lk);
      }
    }
  };
  auto store_tile = [&](int at, bool safe) {
    pq.template store<Dm::PX>(sq[at], safe, flag[at]);
    pg.template store<Dm::PX>(sg[at], safe, flag[at]);
    if (threadIdx.x < RR_XA_KT) { sl[at][threadIdx.x] = nl; sd[at][threadIdx.x] = nd; }
    if (a.mask != nullptr) {
#pragma unroll
      for (int c = 0; c < 4 * KW; c += 4) {                              // four rows by four keys, turned over
        const uint32_t lo0 = __builtin_amdgcn_perm(nm[c + 1], nm[c], 0x05010400), hi0 = __builtin_amdgcn_perm(nm[c + 1], nm[c], 0x07030602);
        const uint32_t lo1 = __builtin_amdgcn_perm(nm[c + 3], nm[c + 2], 0x05010400), hi1 = __builtin_amdgcn_perm(nm[c + 3], nm[c + 2], 0x07030602);
        const uint32_t k4[4] = {__builtin_amdgcn_perm(lo1, lo0, 0x05040100), __builtin_amdgcn_perm(lo1, lo0, 0x07060302), __builtin_amdgcn_perm(hi1, hi0, 0x05040100),
                                __builtin_amdgcn_perm(hi1, hi0, 0x07060302)};
        const int r = mrow + c / 4 * (256 / (4 * KW)), key = threadIdx.x % (16 * KW) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&sm[at][(key + e) * MP + r]) = k4[e];
      }
    }
  };
  if (first < last) load_tile(first);
  typename M::Frag kf[KW][Dm::NK], vf[KW][Dm::NK];
#pragma unroll
  for (int t = 0; t < KW; ++t) {
    const int key = key0 + 16 * t + j;
#pragma unroll
    for (int k = 0; k < Dm::NK; ++k) {
      const int c = k * M::KC + g * M::EPC;
      const bool in = key < seen && c < a.D;
      kf[t][k] = in ? frag_at<T>(kp + (long long)key * a.kl + c) : frag_zero<T>();
      vf[t][k] = in ? frag_at<T>(vp + (long long)key * a.vl + c) : frag_zero<T>();
    }
  }
  f32x4 ok[KW][Dm::DT], ov[KW][Dm::DT];
  float up[KW];                                                          // ds is collected times up 2^14
  // one staged tile of rows.  Rows behind the last one are zeros with an lse of infinity: their weights are zero.  Keys behind the last one hold zeros; what
  // they collect is not written
  auto tile = [&](auto safe, int rows, int at) {
    const T *tq = sq[at], *tg = sg[at];
    const uint32_t* fl = flag[at];
    const bool some = a.mask != nullptr || safe();      // (uniform)
#pragma unroll STEPS
    for (int n = 0; n < 4; n += M::PT) {
      if (SKIP && 16 * n >= rows) break;
      f32x4 s[KW][M::PT], dp[KW][M::PT];
#pragma unroll
      for (int u = 0; u < M::PT; ++u) {
#pragma unroll
        for (int t = 0; t < KW; ++t) { s[t][u] = rr_zero4(); dp[t][u] = rr_zero4(); }
#pragma unroll
        for (int k = 0; k < Dm::NK; ++k) {
          const typename M::Frag fq = frag_at<T>(tq + (16 * (n + u) + j) * Dm::PX + k * M::KC + g * M::EPC);
          const typename M::Frag fg = frag_at<T>(tg + (16 * (n + u) + j) * Dm::PX + k * M::KC + g * M::EPC);
#pragma unroll
          for (int t = 0; t < KW; ++t) { s[t][u] = M::mma(fq, kf[t][k], s[t][u]); dp[t][u] = M::mma(fg, vf[t][k], dp[t][u]); }
        }
        in_order<TIGHT>();
      }
      f32x4 ls[M::PT], de[M::PT];
#pragma unroll
      for (int u = 0; u < M::PT; ++u) {
        ls[u] = *reinterpret_cast<const f32x4*>(&sl[at][16 * (n + u) + 4 * g]);
        de[u] = *reinterpret_cast<const f32x4*>(&sd[at][16 * (n + u) + 4 * g]);
      }
      typename M::Frag pf[KW], df[KW], dr[KW];
#pragma unroll
      for (int t = 0; t < KW; ++t) {
#pragma unroll
        for (int u = 0; u < M::PT; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[t][u][i], c2, -ls[u][i]));
            dp[t][u][i] = p * (Scaled<T>::v ? (dp[t][u][i] - de[u][i]) * up[t] : dp[t][u][i] - de[u][i]);
            s[t][u][i] = p;
          }
        if (some) {
          const int key = key0 + 16 * t + j;
#pragma unroll
          for (int u = 0; u < M::PT; ++u) {
            const int rr = 16 * (n + u) + 4 * g;                     // rows of the tile
            uint32_t b = a.mask != nullptr ? *reinterpret_cast<const uint32_t*>(&sm[at][(key - block0) * MP + rr]) : 0x01010101u;
            b = key < seen ? first_bytes(b, rows - rr) : 0u;
            if constexpr (safe()) {                                              // a row that holds a non-finite value
              const uint32_t fine = ~(flag4(fl, rr) * 0xffu);
              keep4(s[t][u], fine, __builtin_nanf(""));
              keep4(dp[t][u], fine, __builtin_nanf(""));
            }
            keep4(s[t][u], b, 0.f);
            keep4(dp[t][u], b, 0.f);
          }
        }
        pf[t] = M::pack(s[t]);
        if constexpr (Scaled<T>::v) {
          const float mx = abs4(abs4(0.f, dp[t][0]), dp[t][M::PT - 1]);
          if (__any(mx > 32768.f && key0 + 16 * t + j < seen)) {
            const float r = fall_by(group_max(mx));
            up[t] *= r;
#pragma unroll
            for (int u = 0; u < M::PT; ++u) dp[t][u] *= r;
#pragma unroll
            for (int d = 0; d < Dm::DT; ++d) ok[t][d] *= r;
          }
        }
        df[t] = M::pack(dp[t]);
        if constexpr (sizeof(T) == 2) dr[t] = rest_of<T>(dp[t], df[t]);
      }
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) {
        const typename M::Frag fg = M::tr(tg, Dm::PX, 16 * n, 16 * d, lane);
        const typename M::Frag fq = M::tr(tq, Dm::PX, 16 * n, 16 * d, lane);
#pragma unroll
        for (int t = 0; t < KW; ++t) {
          ov[t][d] = M::mma(fg, pf[t], ov[t][d]);
          ok[t][d] = M::mma(fq, df[t], ok[t][d]);
          if constexpr (sizeof(T) == 2) ok[t][d] = M::mma(fq, dr[t], ok[t][d]);
        }
        if ((d & 1) == 1) in_order<TIGHT>();
      }
    }
  };
  auto walk = [&](auto safe) {
#pragma unroll
    for (int t = 0; t < KW; ++t) {
      up[t] = RR_XA_UP / (1 << RR_XA_P_BITS);
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d) { ok[t][d] = rr_zero4(); ov[t][d] = rr_zero4(); }
    }
    if constexpr (safe()) {
      clear_flag(flag[0]);
      load_tile(first);
    }
    if (first < last) store_tile(0, safe());
    __syncthreads();
    int at = 0;
    for (int i = first; i < last; ++i, at ^= 1) {
      const bool more = i + 1 < last;
      if (more) load_tile(i + 1);
      if (busy) tile(safe, a.Lq - i % per_head * RR_XA_KT, at);
      if (more) {
        if constexpr (safe()) clear_flag(flag[at ^ 1]);
        store_tile(at ^ 1, safe());
      }
      __syncthreads();
    }
    bool bad = false;
#pragma unroll
    for (int t = 0; t < KW; ++t)
#pragma unroll
      for (int d = 0; d < Dm::DT; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) bad |= key0 + 16 * t + j < seen && (is_bad(ok[t][d][i]) || is_bad(ov[t][d][i]));
    return __syncthreads_or(bad && busy);
  };
  if (walk(std::false_type{})) walk(std::true_type{});
#pragma unroll
  for (int t = 0; t < KW; ++t) {
    const int key = key0 + 16 * t + j;
    if (key >= a.Lk) continue;
    const long long at_out = (((long long)w.b * a.Lk + key) * a.Hk + w.hk) * a.D;
    const long long half = (long long)a.B * a.Lk * a.Hk * a.D;
    float* p = a.part + (long long)w.split * 2 * half + at_out;
#pragma unroll
    for (int d = 0; d < Dm::DT; ++d) {
      const int c = 16 * d + 4 * g;
      if (c >= a.D) continue;
      const float down = Scaled<T>::v ? 1.f / (1 << RR_XA_P_BITS) : 1.f;
      const f32x4 zero = rr_zero4(), xk = key < seen ? (Scaled<T>::v ? ok[t][d] * (down / up[t]) : ok[t][d]) * a.scale : zero, xv = key < seen ? ov[t][d] * down : zero;
      if (a.nsplit > 1) {
        *reinterpret_cast<f32x4*>(p + c) = xk;
        *reinterpret_cast<f32x4*>(p + half + c) = xv;
      } else {
        typedef T V4 __attribute__((ext_vector_type(4)));
        V4 vk, vv;
#pragma unroll
        for (int i = 0; i < 4; ++i) { vk[i] = (T)xk[i]; vv[i] = (T)xv[i]; }
        *reinterpret_cast<V4*>((T*)a.dk + at_out + c) = vk;
        *reinterpret_cast<V4*>((T*)a.dv + at_out + c) = vv;
      }
    }
  }
}

// adds the splits' partial gradients in order: n values each, `stride` floats between the splits
template <typename T>
__global__ __launch_bounds__(256) void k_xattn_add(const float* __restrict__ part, long long stride, int nsplit, T* __restrict__ out, long long n4) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
    f32x4 t = *reinterpret_cast<const f32x4*>(part + 4 * i);
    for (int s = 1; s < nsplit; ++s) t += *reinterpret_cast<const f32x4*>(part + s * stride + 4 * i);
    typedef T V4 __attribute__((ext_vector_type(4)));
    V4 v;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (T)t[e];
    *reinterpret_cast<V4*>(out + 4 * i) = v;
  }
}

// ------------------------------------------------------------------------------------------------ host
int head_pad(int D) { return D <= 16 ? 16 : D <= 32 ? 32 : D <= 64 ? 64 : 128; }

// rows (or keys) of a workgroup: 4 waves of 16 or 32
struct Plan { int wide, nblk, nsplit, tiles_per_split; };
Plan plan_for(long long kept, long long walked, long long outer, bool narrow) {
  Plan p;
  // 16-bit types: with 16 rows a wave the reads of the staged tiles take LDS twice as long as the products take the matrix pipe, with 32 as long.
  // float32 products are eight times slower: 16 rows, more waves (512 x 8 heads of 100 queries on 100 keys: 66 us, 68 with 32)
  p.wide = !narrow && kept > 64 ? 2 : 1;
  p.nblk = (int)((kept + 64 * p.wide - 1) / (64 * p.wide));
  const long long tiles = (walked + RR_XA_KT - 1) / RR_XA_KT;
  const long long blocks = outer * p.nblk;
  // fewer workgroups than CUs: the walked axis is split, four tiles a split at the least.  A workgroup of many rows writes much for the joining
  // launch: two for each CU; one of few rows hardly any: eight, which also evens out ragged lengths.  With and without the split: one token, 16 / 4 heads of 128, 8 192 keys,
  // 48 sequences 176 / 286 us, 4 sequences 30 / 210; 512 queries on 4 096 keys, 8 heads of 64, 2 sequences 32 / 78, 4 sequences 41 / 101; float32 on 1 024 keys 34 / 57
  const long long target = kept > 64 ? 512 : 2048;
  long long split = blocks >= (kept > 64 ? 256 : 512) ? 1 : (target + blocks - 1) / blocks;
  if (split > tiles / 4) split = tiles / 4;
  if (split < 1) split = 1;
  if (split > 256) split = 256;
  p.tiles_per_split = (int)((tiles + split - 1) / split);
  if (p.tiles_per_split < 1) p.tiles_per_split = 1;
  p.nsplit = (int)((tiles + p.tiles_per_split - 1) / p.tiles_per_split);
  if (p.nsplit < 1) p.nsplit = 1;
  return p;
}

// a launch holds fewer than 2^32 threads: as many batch entries at a time as that allows (one at the least: sizes_of)
#define RR_XA_GRID (0x7fffffffLL / 256)
template <typename F>
void by_launches(XAttn& a, const Plan& p, F launch) {
  a.nsplit = p.nsplit; a.tiles_per_split = p.tiles_per_split; a.nblk = p.nblk;
  const long long each = (long long)a.Hk * p.nsplit * p.nblk, most = RR_XA_GRID / each;
  for (long long b = 0; b < a.B; b += most) {
    a.b0 = (int)b;
    launch(dim3((unsigned)((a.B - b < most ? a.B - b : most) * each)));
  }
}
template <typename T, int DP>
int fwd_go(XAttn& a, const Plan& p, hipStream_t st) {
  by_launches(a, p, [&](dim3 grid) {
    if constexpr (sizeof(T) == 2) {
      if (p.wide == 2) hipLaunchKernelGGL((k_xattn_fwd<T, DP, 2>), grid, dim3(256), 0, st, a);
    }
    if (p.wide == 1) hipLaunchKernelGGL((k_xattn_fwd<T, DP, 1>), grid, dim3(256), 0, st, a);
  });
  if (p.nsplit > 1) hipLaunchKernelGGL((k_xattn_join<T, DP>), dim3((unsigned)(((long long)a.B * a.Hk * a.G * a.Lq + 1024 / DP - 1) / (1024 / DP))), dim3(256), 0, st, a);
  return rr_check(hipGetLastError());
}
template <typename T, int DP>
int bwd_go(XAttn& a, const Plan& p, const Plan& pk, hipStream_t st) {
  by_launches(a, p, [&](dim3 grid) {
    if constexpr (sizeof(T) == 2) {
      if (a.Lk <= RR_XA_KT) {
        if constexpr (DP < 128) {
          if (p.wide == 2) hipLaunchKernelGGL((k_xattn_dq<T, DP, 2, true>), grid, dim3(256), 0, st, a);
        }
        if (p.wide == 1) hipLaunchKernelGGL((k_xattn_dq<T, DP, 1, true>), grid, dim3(256), 0, st, a);
      } else if (p.wide == 2) hipLaunchKernelGGL((k_xattn_dq<T, DP, 2, false>), grid, dim3(256), 0, st, a);
      else hipLaunchKernelGGL((k_xattn_dq<T, DP, 1, false>), grid, dim3(256), 0, st, a);
    } else {
      hipLaunchKernelGGL((k_xattn_dq<T, DP, 1, false>), grid, dim3(256), 0, st, a);
    }
  });
  const long long nq4 = (long long)a.B * a.Lq * a.Hk * a.G * a.D / 4, nk4 = (long long)a.B * a.Lk * a.Hk * a.D / 4;
  auto blocks = [](long long n) { return dim3((unsigned)(n / 256 + 1 < 4096 ? n / 256 + 1 : 4096)); };
  if (p.nsplit > 1) hipLaunchKernelGGL((k_xattn_add<T>), blocks(nq4), dim3(256), 0, st, a.part, 4 * nq4, p.nsplit, (T*)a.dq, nq4);
  by_launches(a, pk, [&](dim3 grid) {
    if constexpr (sizeof(T) == 2) {
      if (pk.wide == 2) hipLaunchKernelGGL((k_xattn_dkv<T, DP, 2>), grid, dim3(256), 0, st, a);
    }
    if (pk.wide == 1) hipLaunchKernelGGL((k_xattn_dkv<T, DP, 1>), grid, dim3(256), 0, st, a);
  });
  if (pk.nsplit > 1) {
    hipLaunchKernelGGL((k_xattn_add<T>), blocks(nk4), dim3(256), 0, st, a.part, 8 * nk4, pk.nsplit, (T*)a.dk, nk4);
    hipLaunchKernelGGL((k_xattn_add<T>), blocks(nk4), dim3(256), 0, st, a.part + 4 * nk4, 8 * nk4, pk.nsplit, (T*)a.dv, nk4);
  }
  return rr_check(hipGetLastError());
}

struct Sizes { Plan q, dq, k; size_t fwd, bwd; bool ok; };
Sizes sizes_of(long long B, long long Lq, long long Lk, long long Hk, long long G, int D, int dtype) {
  Sizes s{};
  const long long lim = 0x7fffffffLL;
  // counts that index rows, keys and workgroups are 32-bit (the last split's end may pass Lk by a tile a split); offsets into the tensors are 64-bit
  s.ok = B >= 1 && Lq >= 1 && Lk >= 0 && Hk >= 1 && G >= 1 && D >= 8 && D <= 128 && D % 8 == 0 && Lq <= lim && Lk <= lim - 65536 && G * (Lq + 64) <= lim - 256 && B <= lim && Hk <= lim &&
         B * Hk <= lim && G * Hk <= lim;
  if (!s.ok) return s;
  s.q = plan_for(G * Lq, Lk, B * Hk, dtype == RR_F32);
  s.k = plan_for(Lk > 0 ? Lk : 1, G * ((Lq + RR_XA_KT - 1) / RR_XA_KT) * RR_XA_KT, B * Hk, dtype == RR_F32);
  // dq of 128 columns on keys of one tile holds too much for 32 rows a wave without spilling: 120 queries on 60 keys, 2 048 heads, 182 us spilling, 132 with one
  // workgroup a CU, 97 with 16 rows a wave
  s.dq = plan_for(G * Lq, Lk, B * Hk, dtype == RR_F32 || (D > 64 && Lk <= RR_XA_KT));
  auto fits = [&](const Plan& p) { return Hk * p.nsplit * p.nblk <= RR_XA_GRID; };
  if (!fits(s.q) || !fits(s.dq) || !fits(s.k) || B * Hk * G * Lq > lim) { s.ok = false; return s; }
  const int DP = head_pad(D);
  s.fwd = s.q.nsplit > 1 ? (size_t)(B * Hk * G * Lq) * s.q.nsplit * RR_XA_PART(DP) * 4 : 0;
  const size_t b1 = s.dq.nsplit > 1 ? (size_t)s.dq.nsplit * B * Lq * Hk * G * D * 4 : 0, b2 = s.k.nsplit > 1 ? (size_t)s.k.nsplit * 2 * B * Lk * Hk * D * 4 : 0;
  s.bwd = b1 > b2 ? b1 : b2;
  return s;
}

bool well_placed(const void* p, long long sb, long long sl, long long sh, int size) {
  const int e = 16 / size;
  return p != nullptr && rr_aligned16(p) && sb % e == 0 && sl % e == 0 && sh % e == 0;
}

}  // namespace

static int xa_fill(const XAttnIO* io, XAttn& a, bool bwd) {
  const int size = io->dtype == RR_F32 ? 4 : 2;
  a = {};
  if (io->dtype < 0 || io->dtype > 2 || !(io->scale > 0.f) || io->scale > 3.0e38f) return RR_EINVAL;
  if (io->Lk > 0 && (!well_placed(io->k, io->k_stride[0], io->k_stride[1], io->k_stride[2], size) || !well_placed(io->v, io->v_stride[0], io->v_stride[1], io->v_stride[2], size)))
    return RR_EINVAL;
  if (!well_placed(io->q, io->q_stride[0], io->q_stride[1], io->q_stride[2], size) || io->out == nullptr || !rr_aligned16(io->out)) return RR_EINVAL;
  if (bwd && (!well_placed(io->dout, io->dout_stride[0], io->dout_stride[1], io->dout_stride[2], size) || io->lse == nullptr || io->delta == nullptr ||
              !rr_aligned16(io->dq) || !rr_aligned16(io->dk) || !rr_aligned16(io->dv) || io->dq == nullptr || (io->Lk > 0 && (io->dk == nullptr || io->dv == nullptr))))
    return RR_EINVAL;
  a.q = io->q; a.k = io->k; a.v = io->v; a.out = io->out; a.lse = io->lse; a.mask = io->mask; a.lens = io->kv_lens;
  a.qb = io->q_stride[0]; a.ql = io->q_stride[1]; a.qh = io->q_stride[2];
  a.kb = io->k_stride[0]; a.kl = io->k_stride[1]; a.kh = io->k_stride[2];
  a.vb = io->v_stride[0]; a.vl = io->v_stride[1]; a.vh = io->v_stride[2];
  a.mb = io->mask_stride[0]; a.mh = io->mask_stride[1]; a.ml = io->mask_stride[2];
  a.gb = io->dout_stride[0]; a.gl = io->dout_stride[1]; a.gh = io->dout_stride[2];
  a.lens64 = io->lens_int64; a.B = io->B; a.Lq = io->Lq; a.Lk = io->Lk; a.Hk = io->Hk; a.G = io->G; a.D = io->D;
  a.scale = io->scale; a.part = (float*)io->workspace; a.dout = io->dout; a.delta = io->delta; a.dq = io->dq; a.dk = io->dk; a.dv = io->dv;
  return RR_OK;
}

extern "C" long long rr_cross_attn_workspace(int dtype, int B, int Lq, int Lk, int Hk, int G, int D, int backward) {
  const Sizes s = sizes_of(B, Lq, Lk, Hk, G, D, dtype);
  return s.ok ? (long long)(backward ? s.bwd : s.fwd) : -1;
}

#define RR_XA_BY_DIM(T, CALL)                                   \
  switch (head_pad(io->D)) {                                    \
    case 16: { constexpr int DP = 16; return CALL(T, DP); }     \
    case 32: { constexpr int DP = 32; return CALL(T, DP); }     \
    case 64: { constexpr int DP = 64; return CALL(T, DP); }     \
    default: { constexpr int DP = 128; return CALL(T, DP); }    \
  }

extern "C" int rr_cross_attn(const XAttnIO* io, hipStream_t st) {
  if (io == nullptr) return RR_EINVAL;
  const Sizes s = sizes_of(io->B, io->Lq, io->Lk, io->Hk, io->G, io->D, io->dtype);
  XAttn a;
  if (!s.ok || xa_fill(io, a, false) != RR_OK || (s.fwd > 0 && (io->workspace == nullptr || (size_t)io->workspace_bytes < s.fwd || !rr_aligned16(io->workspace)))) return RR_EINVAL;
#define RR_CALL(T, DP) fwd_go<T, DP>(a, s.q, st)
  if (io->dtype == RR_F32) { RR_XA_BY_DIM(float, RR_CALL) }
  if (io->dtype == RR_F16) { RR_XA_BY_DIM(rr_f16, RR_CALL) }
  RR_XA_BY_DIM(rr_bf16, RR_CALL)
#undef RR_CALL
}

extern "C" int rr_cross_attn_bwd(const XAttnIO* io, hipStream_t st) {
  if (io == nullptr || io->Lk < 1) return RR_EINVAL;
  const Sizes s = sizes_of(io->B, io->Lq, io->Lk, io->Hk, io->G, io->D, io->dtype);
  XAttn a;
  if (!s.ok || xa_fill(io, a, true) != RR_OK || (s.bwd > 0 && (io->workspace == nullptr || (size_t)io->workspace_bytes < s.bwd || !rr_aligned16(io->workspace)))) return RR_EINVAL;
#define RR_CALL(T, DP) bwd_go<T, DP>(a, s.dq, s.k, st)
  if (io->dtype == RR_F32) { RR_XA_BY_DIM(float, RR_CALL) }
  if (io->dtype == RR_F16) { RR_XA_BY_DIM(rr_f16, RR_CALL) }
  RR_XA_BY_DIM(rr_bf16, RR_CALL)
#undef RR_CALL
}
