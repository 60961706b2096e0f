// One choice a row from logits with a given random number: temperature, top-k, top-p and min-p filters, inverse CDF
// (process_logits + sampling of rrnco/models/decoding.py:37-63, 272-298, 311-361 with min-p and the random numbers as an input).
//
//   z_i = l_i / T,  w_i = exp(z_i - max z);  keys that are masked, NaN or -inf take no part
//   top-k   keeps l >= the k-th largest (copies of it too: equal logits stay or go together)
//   top-p   of those, keeps every key with less than p of their mass strictly above it
//   min-p   keeps w_i >= min_p (the largest weight is 1)
//   choice  the first index i, in index order, with sum_{j <= i} w_j > u sum_j w_j;  logp = log(w_i / sum w)
//
// A border decided wrongly changes a whole number, so weights and their sums are held in 64 bits: a sum of V weights in 32 bits
// moves each of the V borders of the CDF by 1e-7 and draws another key for about V * 1e-7 of the random numbers.  Thresholds are
// found among the logits' ordered bit patterns, exactly; nothing is sorted.
//
// Up to 1 024 keys: a wave a row, its keys in registers.  The k-th largest by bisection over the bit patterns that the row's extremes
// leave open (one ballot a register and step); what it keeps, where it fits one register a lane, moves together, in index order, so that
// only kept keys pay for their 64-bit weight.  Longer rows: a workgroup a row, its keys in registers up to 16 384: a histogram over the
// distance from the maximum, then only the keys of the bin that holds the border are looked at.  Masses there are whole numbers of steps
// of 2^-45, so that atomics may add them in any order; sums over more than 2^18 keys may pass 64 bits and are kept in 128.  Longer rows: a workgroup for every 16 384 keys, five
// launches (below).
// Bound by vector instructions, not by the one read of the logits: 51 200 x 100 float32 with a mask 17 us (1.5 TB/s), 762 of them a wave of four rows, 95 for each key that a lane holds, of
// which its 64-bit weight is some 20: the rest are keys and masks, comparisons and selects in 64 bits, the scans and the logarithm.  4 096 x 1 001 with all filters 23 us, the
// bisections' dependent steps; 64 x 131 072 bf16 with settings of each row 79 - 88 us in five launches (6 + 16 + 7 + 13 + 28).
#include <type_traits>

#include "rr_types.h"

namespace {

struct Draw {
  const void* logits;
  const uint8_t* mask;                 // [R][V] by row stride, 1 = may be drawn, or NULL
  const float* u;
  int64_t* index;
  float* logp;
  const float *pt, *pp, *pm;           // per-row temperature, top_p, min_p, or NULL: the scalars
  const int* pk;
  double t, c2, p, mp;
  long long ld, ldm;
  int k, R, V;
};

struct Par { double t, c2, p, mp, u; int k; bool greedy; };
__device__ __forceinline__ Par par_of(const Draw& a, int r) {
  Par q;
  const double t = a.pt ? (double)a.pt[r] : a.t;
  q.greedy = !(t > 0.0);                                       // 0 (and whatever is no temperature): the largest logit
  q.t = t;
  q.c2 = a.pt ? 1.44269504088896340736 / t : a.c2;                           // weight of a key: 2^((l - max) c2)
  q.k = a.pk ? a.pk[r] : a.k;
  q.p = a.pp ? (double)a.pp[r] : a.p;
  q.mp = a.pm ? (double)a.pm[r] : a.mp;
  q.mp = q.mp > 1.0 ? 1.0 : q.mp;                              // the largest weight is 1: something is always left
  const double u = (double)a.u[r];
  q.u = u > 0.0 ? (u < 1.0 ? u : 0.99999999999999989) : 0.0;   // a number outside [0, 1) counts as the nearer end, NaN as 0
  return q;
}

__device__ __forceinline__ uint32_t key_of(float l, bool ok) {           // ordered bit pattern, 0: takes no part
  const uint32_t b = __float_as_uint(l + 0.0f);                          // (-0 counts as 0)
  const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
  return ok && l == l && k > 0x007fffffu ? k : 0u;
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k); }
__device__ __forceinline__ double z_of(uint32_t k, uint32_t top, double c2) { return k == top ? 0.0 : ((double)value_of(k) - (double)value_of(top)) * (c2 * 0.69314718055994530942); }
__device__ __forceinline__ double pow2_of(double f) {
  double p = 4.4455382718708109e-10;
  p = fma(p, f, 7.0549116208011225e-09);
  p = fma(p, f, 1.0178086009239699e-07);
  p = fma(p, f, 1.3215486790144307e-06);
  p = fma(p, f, 1.5252733804059841e-05);
  p = fma(p, f, 1.5403530393381608e-04);
  p = fma(p, f, 1.3333558146428443e-03);
  p = fma(p, f, 9.6181291076284769e-03);
  p = fma(p, f, 5.5504108664821576e-02);
  p = fma(p, f, 2.4022650695910069e-01);
  p = fma(p, f, 6.9314718055994529e-01);
  return fma(p, f, 1.0);
}
// w = 2^((l - max) c2) to 1e-14: the exponent's nearest whole number goes to ldexp, 2^f on [-1/2, 1/2] is its Taylor series (ln 2)^n / n! f^n up to
// n = 11 (the next term is 6e-15).  About 20 instructions; the library's exp with the division by T took three times that.
__device__ __forceinline__ double weight_of(uint32_t k, uint32_t top, double topd, double c2) {
  double t = ((double)value_of(k) - topd) * c2;
  t = t > -2000.0 ? t : -2000.0;                               // under the smallest number: 0, also for what an infinite maximum leaves
  const double n = __builtin_rint(t);
  const double w = ldexp(pow2_of(t - n), (int)n);
  return k == top ? 1.0 : w;
}

// ---- wave helpers on DPP: 16-lane rows by shifts, rows joined by broadcasts; lane 63 then holds the whole wave
#define RR_DPP(v, old, ctrl, rows) __builtin_amdgcn_update_dpp((int)(old), (int)(v), ctrl, rows, 0xf, false)
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_d(double v) {                      // 0 where there is no source lane
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)RR_DPP((uint32_t)b, 0, CTRL, ROWS), hi = (uint32_t)RR_DPP((uint32_t)(b >> 32), 0, CTRL, ROWS);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan_d(double v) {                // inclusive
  v += dpp_d<0x111, 0xf>(v);
  v += dpp_d<0x112, 0xf>(v);
  v += dpp_d<0x114, 0xf>(v);
  v += dpp_d<0x118, 0xf>(v);
  v += dpp_d<0x142, 0xa>(v);
  v += dpp_d<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ double last_lane_d(double v) {
  const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, 63), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), 63);
  return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_d(double v) { return last_lane_d(wave_scan_d(v)); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) { const uint32_t x = (uint32_t)RR_DPP(v, 0, CTRL, ROWS); return v > x ? v : x; }
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
  v = dpp_max<0x111, 0xf>(v);
  v = dpp_max<0x112, 0xf>(v);
  v = dpp_max<0x114, 0xf>(v);
  v = dpp_max<0x118, 0xf>(v);
  v = dpp_max<0x142, 0xa>(v);
  v = dpp_max<0x143, 0xc>(v);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint32_t wave_min_u(uint32_t v) { return ~wave_max_u(~v); }

// log(x), x >= 1: the 32-bit logarithm is off by less than 1e-6 and one step x e^-y - 1 = d, log x = y + d - d^2 / 2, leaves d^3 / 3
__device__ __forceinline__ double log_of(double x) {
  const double y2 = (double)__log2f((float)x);
  const double n = __builtin_rint(y2), f = n - y2;
  const double d = fma(x, ldexp(pow2_of(f), -(int)n), -1.0);
  return y2 * 0.69314718055994530942 + (d - 0.5 * d * d);
}

__device__ __forceinline__ double wave_total(double v) { return wave_sum_d(v); }
__device__ __forceinline__ uint32_t wave_total(uint32_t v) {
#define RR_ADD(CTRL, ROWS) v += (uint32_t)RR_DPP(v, 0, CTRL, ROWS)
  RR_ADD(0x111, 0xf); RR_ADD(0x112, 0xf); RR_ADD(0x114, 0xf); RR_ADD(0x118, 0xf); RR_ADD(0x142, 0xa); RR_ADD(0x143, 0xc);
#undef RR_ADD
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ unsigned long long wave_total(unsigned long long v) {
#define RR_ADD(CTRL, ROWS) v += (unsigned long long)(uint32_t)RR_DPP((uint32_t)(v >> 32), 0, CTRL, ROWS) << 32 | (uint32_t)RR_DPP((uint32_t)v, 0, CTRL, ROWS)
  RR_ADD(0x111, 0xf); RR_ADD(0x112, 0xf); RR_ADD(0x114, 0xf); RR_ADD(0x118, 0xf); RR_ADD(0x142, 0xa); RR_ADD(0x143, 0xc);
#undef RR_ADD
  return (unsigned long long)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
typedef unsigned __int128 rr_u128;
__device__ __forceinline__ unsigned long long hi_of(rr_u128 v) { return (unsigned long long)(v >> 64); }
__device__ __forceinline__ rr_u128 wave_total(rr_u128 v) {
#define RR_WORD(W, CTRL, ROWS) (rr_u128)(uint32_t)RR_DPP((uint32_t)(v >> (32 * W)), 0, CTRL, ROWS) << (32 * W)
#define RR_ADD(CTRL, ROWS) v += RR_WORD(3, CTRL, ROWS) | RR_WORD(2, CTRL, ROWS) | RR_WORD(1, CTRL, ROWS) | RR_WORD(0, CTRL, ROWS)
  RR_ADD(0x111, 0xf); RR_ADD(0x112, 0xf); RR_ADD(0x114, 0xf); RR_ADD(0x118, 0xf); RR_ADD(0x142, 0xa); RR_ADD(0x143, 0xc);
#undef RR_ADD
#undef RR_WORD
  rr_u128 t = 0;
#pragma unroll
  for (int w = 3; w >= 0; --w) t = t << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> (32 * w)), 63);
  return t;
}
// sums as 64-bit floats: never falling in the sum, which is all that the comparisons with a limit need
__device__ __forceinline__ double float_of(uint32_t v) { return (double)v; }
__device__ __forceinline__ double float_of(unsigned long long v) { return (double)v; }
__device__ __forceinline__ double float_of(rr_u128 v) { return (double)hi_of(v) * 18446744073709551616.0 + (double)(unsigned long long)v; }
template <typename V>
__device__ __forceinline__ V lanes_up(V v, int o) {
  if constexpr (sizeof(V) == 16) return (rr_u128)__shfl_up(hi_of(v), o) << 64 | __shfl_up((unsigned long long)v, o);
  else return __shfl_up(v, o);
}
__device__ __forceinline__ void wave_lds() {                             // LDS written by a lane of this wave may be read by another from here on
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

template <int E>
__device__ __forceinline__ int count_ge(const uint32_t (&key)[E], uint32_t at) {
  int n = 0;
#pragma unroll
  for (int q = 0; q < E; ++q) n += __popcll(__ballot(key[q] >= at));
  return n;
}
// a bit pattern between two (lo < hi, both of finite values), by value: halving patterns would spend its steps on the exponents around zero
__device__ __forceinline__ uint32_t between(uint32_t lo, uint32_t hi, int step) {
  const uint32_t half = lo + ((hi - lo) >> 1);
  const uint32_t k = key_of(0.5f * value_of(lo) + 0.5f * value_of(hi), true);
  return (step & 3) == 3 || k < lo || k >= hi ? half : k;                // (every fourth by pattern: at most 4 x 32 steps whatever the values)
}

// the k-th largest of the wave's keys (k <= their number), top = the largest
template <int E>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[E], int k, uint32_t top) {
  uint32_t low = top;
#pragma unroll
  for (int q = 0; q < E; ++q) low = key[q] && key[q] < low ? key[q] : low;
  low = wave_min_u(low);
  uint32_t lo = low, hi = top;                                           // count(>= lo) >= k always holds; hi: the answer is <= hi
  for (int step = 0; lo < hi; ++step) {
    const uint32_t mid = between(lo, hi, step) + 1u;
    const int n = count_ge(key, mid);
    if (n >= k) lo = mid; else hi = mid - 1u;
    if (n == k) {                                                        // exactly k keys from mid on: the smallest of them
      uint32_t v = 0xffffffffu;
#pragma unroll
      for (int q = 0; q < E; ++q) v = key[q] >= mid && key[q] < v ? key[q] : v;
      return wave_min_u(v);
    }
  }
  return lo;
}

// The threshold of top-p among a wave's keys and weights: the smallest value with less than `lim` of mass strictly above it, `above` of which is
// outside these keys (all larger).  Weights of 64-bit floats or of whole steps.
template <int E, typename W>
__device__ __forceinline__ uint32_t mass_threshold(const uint32_t (&key)[E], const W (&w)[E], uint32_t top, double above, double lim, uint32_t* skey, W* sw, int lane) {
  uint32_t low = top;
#pragma unroll
  for (int e = 0; e < E; ++e) low = key[e] && key[e] < low ? key[e] : low;
  uint32_t lo = wave_min_u(low), hi = top;                               // mass(> hi) < lim holds
  for (int step = 0; lo < hi; ++step) {
    const uint32_t mid = between(lo, hi, step);
    W m = 0;
    int n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m += key[e] > mid ? w[e] : W(0);
    if (above + (double)wave_total(m) < lim) hi = mid; else lo = mid + 1u;
    // one value between the ends: the next key from lo on is the threshold
#pragma unroll
    for (int e = 0; e < E; ++e) n += __popcll(__ballot(key[e] >= lo && key[e] <= hi));
    if (n <= 1) break;
    if constexpr (E > 1) {
      if (n <= 64) {                                                     // few left: one a lane, what lies above them is summed once
        W over = 0;
        int base = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const bool in = key[e] >= lo && key[e] <= hi;
          const unsigned long long b = __ballot(in);
          const int at = base + __popcll(b & ((1ull << lane) - 1ull));
          if (in) { skey[at] = key[e]; sw[at] = w[e]; }
          base += __popcll(b);
          over += key[e] > hi ? w[e] : W(0);
        }
        wave_lds();
        const uint32_t k1[1] = {lane < n ? skey[lane] : 0u};
        const W w1[1] = {lane < n ? sw[lane] : W(0)};
        wave_lds();
        return mass_threshold<1, W>(k1, w1, wave_max_u(k1[0]), above + (double)wave_total(over), lim, skey, sw, lane);
      }
    }
  }
  return lo;
}

// keys (0: none) of one row in index order: register-major, lane-minor; idx of a register's key; whole: the mass that top-p refers to (below 0: that of these
// keys).  Writes the choice.
template <int E, typename IDX>
__device__ __forceinline__ void choose(const Draw& a, const Par& q, int r, uint32_t (&key)[E], IDX idx, uint32_t top, double whole, uint32_t* skey, double* sw, int lane) {
  const double topd = (double)value_of(top);
  double w[E], z = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = key[e] ? weight_of(key[e], top, topd, q.c2) : 0.0;
    z += w[e];
  }
  if (q.p > 0.0 && q.p < 1.0) {
    const uint32_t lo = mass_threshold<E, double>(key, w, top, 0.0, q.p * (whole < 0.0 ? wave_sum_d(z) : whole), skey, sw, lane);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (key[e] < lo) { key[e] = 0u; w[e] = 0.0; }
  }
  z = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (q.mp > 0.0 && w[e] < q.mp) w[e] = 0.0;
    z += w[e];
  }
  // running sums in index order: two registers are scanned at once; of more, their masses tell the register and only that one is scanned.
  // rounding may leave the target at the very end: then the last key with a weight is taken
  double total = 0.0, cum = 0.0, we = w[0];
  uint32_t ke = key[0];
  int ie = idx(0);
  bool over = false;
  if constexpr (E == 1) {
    cum = wave_scan_d(we);
    total = last_lane_d(cum);
  } else if constexpr (E == 2) {
    const double c0 = wave_scan_d(w[0]), c1 = wave_scan_d(w[1]), t0 = last_lane_d(c0), t1 = last_lane_d(c1);
    total = t0 + t1;
    const bool first = t0 > q.u * total || t1 == 0.0;
    cum = first ? c0 : t0 + c1;
    if (!first) { we = w[1]; ke = key[1]; ie = idx(1); }
  } else {
    double part[E], before = 0.0, base = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) { part[e] = wave_sum_d(w[e]); total += part[e]; }
    int reg = -1, last = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (part[e] > 0.0) last = e;
      if (reg < 0 && before + part[e] > q.u * total) { reg = e; base = before; }
      before += part[e];
    }
    over = reg < 0;
    if (over) reg = last;
#pragma unroll
    for (int e = 1; e < E; ++e)
      if (e == reg) { we = w[e]; ke = key[e]; ie = idx(e); }
    cum = base + wave_scan_d(we);
  }
  const unsigned long long hit = __ballot(!over && we > 0.0 && cum > q.u * total), any = __ballot(we > 0.0);
  const int at = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll((long long)any);
  const float lp = (float)(z_of(ke, top, q.c2) - log_of(total));
  if (lane == at) {
    a.index[r] = ie;
    a.logp[r] = lp;
  }
}

template <typename T, int E>
__global__ __launch_bounds__(256) void k_draw_wave(Draw a) {
  __shared__ uint32_t skey[E > 1 ? 4 : 1][64];
  __shared__ int sidx[E > 1 ? 4 : 1][64];
  __shared__ double sw[E > 1 ? 4 : 1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = blockIdx.x * 4 + wave;      // (the row's addresses in scalar registers)
  if (r >= a.R) return;                                                  // (no workgroup barrier below)
  const T* row = (const T*)a.logits + (long long)r * a.ld;
  uint32_t key[E];
  uint32_t top = 0u;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const int i = lane + 64 * e;
    const bool in = i < a.V;
    const float l = in ? (float)row[i] : 0.f;
    key[e] = key_of(l, in && (a.mask == nullptr || a.mask[(long long)r * a.ldm + (in ? i : 0)] != 0));
    top = key[e] > top ? key[e] : top;
  }
  const Par q = par_of(a, r);
  top = wave_max_u(top);
  if (top == 0u) {                                                       // nothing may be drawn
    if (lane == 0) { a.index[r] = 0; a.logp[r] = -INFINITY; }
    return;
  }
  if (q.greedy) {
    int at = 0x7fffffff;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) {
      const unsigned long long b = __ballot(key[e] == top);
      if (b) at = 64 * e + __ffsll((unsigned long long)b) - 1;
    }
    if (lane == 0) { a.index[r] = at; a.logp[r] = 0.f; }
    return;
  }
  if (q.k > 0 && q.k < a.V && count_ge(key, 1u) > q.k) {
    const uint32_t cut = kth_largest(key, q.k, top);
#pragma unroll
    for (int e = 0; e < E; ++e) key[e] = key[e] >= cut ? key[e] : 0u;
    if constexpr (E > 1) {
      const int n = count_ge(key, 1u);
      if (n <= 64) {                                                     // together, in index order, one a lane
        int base = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const unsigned long long b = __ballot(key[e] != 0u);
          const int at = base + __popcll(b & ((1ull << lane) - 1ull));
          if (key[e]) { skey[wave][at] = key[e]; sidx[wave][at] = lane + 64 * e; }
          base += __popcll(b);
        }
        wave_lds();
        uint32_t k1[1] = {lane < n ? skey[wave][lane] : 0u};
        const int i1 = lane < n ? sidx[wave][lane] : 0;
        choose<1>(a, q, r, k1, [&](int) { return i1; }, top, -1.0, nullptr, nullptr, lane);
        return;
      }
    }
  }
  choose<E>(a, q, r, key, [&](int e) { return lane + 64 * e; }, top, -1.0, skey[E > 1 ? wave : 0], sw[E > 1 ? wave : 0], lane);
}

// ---- short rows without top-k and top-p: 16 lanes a row, E consecutive keys a lane; four rows share every exchange between lanes
template <int CTRL>
__device__ __forceinline__ uint32_t ror_max(uint32_t v) { const uint32_t x = (uint32_t)RR_DPP(v, 0, CTRL, 0xf); return v > x ? v : x; }

template <typename T, int E, bool VECTOR>
__global__ __launch_bounds__(256) void k_draw_group(Draw a) {
  constexpr int VEC = VECTOR ? rr_vec_of<T>::N : 1;
  static_assert(E % VEC == 0, "whole pieces");
  const int lane = threadIdx.x & 15, r = blockIdx.x * 16 + (threadIdx.x >> 4);
  const bool live = r < a.R;
  const int rc = live ? r : a.R - 1;                                     // (a row behind the last one repeats it and writes nothing)
  const T* row = (const T*)a.logits + (long long)rc * a.ld;
  const uint8_t* mask = a.mask != nullptr ? a.mask + (long long)rc * a.ldm : nullptr;
  const int i0 = lane * E;
  uint32_t key[E], top = 0u;
#pragma unroll
  for (int p = 0; p < E; p += VEC) {
    float x[VEC];
    uint8_t m[VEC];
    const bool in = i0 + p < a.V;                                        // (pieces are whole: V is a multiple of VEC)
#pragma unroll
    for (int i = 0; i < VEC; ++i) { x[i] = 0.f; m[i] = 1; }
    if (in) {
      rr_load_n<T, VEC>(row + i0 + p, x);
      if (mask != nullptr) __builtin_memcpy(m, mask + i0 + p, VEC);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) { key[p + i] = key_of(x[i], in && m[i] != 0); top = key[p + i] > top ? key[p + i] : top; }
  }
  top = ror_max<0x128>(top);                                             // row_ror 8, 4, 2, 1: every lane of a row gets its maximum
  top = ror_max<0x124>(top);
  top = ror_max<0x122>(top);
  top = ror_max<0x121>(top);
  const Par q = par_of(a, rc);
  const double topd = (double)value_of(top);
  double w[E], s = 0.0;
  int first = 0x7fffffff;
#pragma unroll
  for (int e = E - 1; e >= 0; --e) first = key[e] == top && top ? i0 + e : first;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = key[e] ? weight_of(key[e], top, topd, q.c2) : 0.0;
    if (w[e] < q.mp) w[e] = 0.0;
    if (q.greedy) w[e] = i0 + e == first ? 1.0 : 0.0;                    // (one a lane; the lowest lane's wins below)
    s += w[e];
  }
  double inc = s;
  inc += dpp_d<0x111, 0xf>(inc);
  inc += dpp_d<0x112, 0xf>(inc);
  inc += dpp_d<0x114, 0xf>(inc);
  inc += dpp_d<0x118, 0xf>(inc);
  const double total = __shfl(inc, (threadIdx.x & 48) | 15);
  const double target = q.greedy ? 0.0 : q.u * total;
  const int shift = threadIdx.x & 48;
  const unsigned hits = (unsigned)(__ballot(s > 0.0 && inc > target) >> shift) & 0xffffu, any = (unsigned)(__ballot(s > 0.0) >> shift) & 0xffffu;
  if (!live) return;
  if (any == 0u) {                                                       // nothing may be drawn
    if (lane == 0) { a.index[r] = 0; a.logp[r] = -INFINITY; }
    return;
  }
  const int at = hits ? __ffs(hits) - 1 : 31 - __clz(any);               // (rounding may leave the target at the very end: the last key with a weight)
  if (lane != at) return;
  double c = inc - s;
  uint32_t k = 0u;
  int pick = 0;
  bool done = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    c += w[e];
    const bool take = w[e] > 0.0 && !done;
    k = take ? key[e] : k;
    pick = take ? i0 + e : pick;
    done = done || (take && hits != 0u && c > target);
  }
  a.index[r] = pick;
  a.logp[r] = q.greedy ? 0.f : (float)(z_of(k, top, q.c2) - log_of(total));
}

// ------------------------------------------------------------------------------------------------ long rows
#define RR_DRAW_BINS 1024
#define RR_DRAW_LIST 2048
#define RR_DRAW_STEP 35184372088832.0          // 2^45 steps a unit of weight
#define RR_DRAW_NT 1024                        // the split form's workgroups, and the keys of its stretches
#define RR_DRAW_STRETCH 16384

// bin of a key: its distance from the maximum in steps of T / 32 (monotone in the key), the last bin open
__device__ __forceinline__ int bin_of(uint32_t k, float topv, float per) {
  const float v = value_of(k), d = (topv - v) * per;
  return d < (float)(RR_DRAW_BINS - 1) ? (int)d : (v == topv ? 0 : RR_DRAW_BINS - 1);
}
__device__ __forceinline__ unsigned long long steps_of(double w) {       // w <= 1: w 2^45 + 2^52 holds the whole number in its low bits
  return __builtin_bit_cast(unsigned long long, fma(w, RR_DRAW_STEP, 4503599627370496.0)) & 0xfffffffffffffull;
}

// E keys a thread of NT * E consecutive ones from `base` on: piece-major, then thread, VEC keys each (index order within each level)
template <typename T, int NT, int E>
struct Keys {
  static constexpr int VEC = rr_vec_of<T>::N, P = E / VEC, N = NT * E;
  uint32_t key[E];
  int base;
  __device__ __forceinline__ int index(int e) const { return base + (e / VEC * NT + (int)threadIdx.x) * VEC + e % VEC; }
  __device__ __forceinline__ void load(const T* row, const uint8_t* mask, int from, int V) {
    base = from;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int i0 = base + (p * NT + (int)threadIdx.x) * VEC;
      if (i0 + VEC <= V) {
        float x[VEC];
        uint8_t m[VEC];
        rr_load_n<T, VEC>(row + i0, x);
#pragma unroll
        for (int i = 0; i < VEC; ++i) m[i] = 1;
        if (mask != nullptr) __builtin_memcpy(m, mask + i0, VEC);
#pragma unroll
        for (int i = 0; i < VEC; ++i) key[p * VEC + i] = key_of(x[i], m[i] != 0);
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) key[p * VEC + i] = i0 + i < V ? key_of((float)row[i0 + i], mask == nullptr || mask[i0 + i] != 0) : 0u;
      }
    }
  }
  template <typename F>
  __device__ __forceinline__ void each(F f) const {
#pragma unroll
    for (int e = 0; e < E; ++e) f(key[e], index(e));
  }
};

template <int NT, typename V>
__device__ __forceinline__ V block_sum(V v, V* red) {                    // every thread gets the sum, added in a fixed order
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  V t = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t += red[i];
  return t;
}
template <int NT>
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* red) {
  v = wave_max_u(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) t = t > red[i] ? t : red[i];
  return t;
}

// the first bin, from the top, at which the running sum of the bins' h reaches `need` (> 0), the last one if none before it does: its number and the sum before it
template <int NT, typename V, typename H>
__device__ __forceinline__ void find_bin(H h, double need, V* red, int* found, V* above) {
  constexpr int PER = RR_DRAW_BINS / NT;
  static_assert(PER >= 1, "a bin for each thread");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = threadIdx.x * PER;
  V mine = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) mine += h(b0 + i);
  V run = mine;                                                          // inclusive over the wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V x = lanes_up(run, o);
    if (lane >= o) run += x;
  }
  __syncthreads();
  if (lane == 63) red[wave] = run;
  if (threadIdx.x == 0) *found = RR_DRAW_BINS - 1;
  __syncthreads();
  V base = run - mine;
  for (int i = 0; i < wave; ++i) base += red[i];
  for (int i = 0; i < PER; ++i) {
    const V next = base + h(b0 + i);
    if (float_of(base) < need && (float_of(next) >= need || b0 + i == RR_DRAW_BINS - 1)) { *found = b0 + i; *above = base; }      // one thread at the most: sums do not fall
    base = next;
  }
  __syncthreads();
}

template <int NT, int LIST>
struct Scratch {
  static constexpr int LISTED = LIST;
  unsigned long long mass[RR_DRAW_BINS];
  uint32_t cnt[RR_DRAW_BINS];
  uint32_t list[LIST];
  double part[512], redd[NT / 64];
  unsigned long long redm[NT / 64], above_m;
  uint32_t redu[NT / 64], above_c;
  int found, nlist;
};

// what the thresholds leave of a key's weight
struct Kept {
  uint32_t top, cut;
  double topd, c2, mp;
  __device__ __forceinline__ double operator()(uint32_t k) const {
    if (k < cut || k == 0u) return 0.0;
    const double w = weight_of(k, top, topd, c2);
    return w < mp ? 0.0 : w;
  }
};

// the choice among the keys of one stretch: `base` is the mass before it, `total` the row's (below 0: this stretch is the row).  Each wave's mass of each
// piece goes to LDS, every wave finds the (piece, wave) that the target falls in, that wave scans its lanes, the lane walks its VEC keys
template <typename T, int NT, int E, typename S>
__device__ __forceinline__ void locate(const Draw& a, const Par& q, int r, const Keys<T, NT, E>& ks, const Kept& kept, double base, double total, S& sh) {
  using K = Keys<T, NT, E>;
  constexpr int NW = NT / 64, N = K::P * NW, PER = (N + 63) / 64;
  static_assert(N <= 512, "the table of parts");
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double s[K::P];
  __syncthreads();
#pragma unroll
  for (int p = 0; p < K::P; ++p) {
    s[p] = 0.0;
#pragma unroll
    for (int i = 0; i < K::VEC; ++i) s[p] += kept(ks.key[p * K::VEC + i]);
    const double t = wave_sum_d(s[p]);
    if (lane == 0) sh.part[p * NW + wave] = t;
  }
  __syncthreads();
  double mine[PER], m = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) { mine[i] = lane * PER + i < N ? sh.part[lane * PER + i] : 0.0; m += mine[i]; }
  double run = wave_scan_d(m);
  if (total < 0.0) { total = last_lane_d(run); base = 0.0; }
  const double target = q.u * total;
  run = base + (run - m);
  int hit = 0x7fffffff, last = -1;
  double before = 0.0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (mine[i] > 0.0) last = lane * PER + i;
    if (hit == 0x7fffffff && mine[i] > 0.0 && run + mine[i] > target) { hit = lane * PER + i; before = run; }
    run += mine[i];
  }
  const unsigned long long hits = __ballot(hit != 0x7fffffff), lasts = __ballot(last >= 0);
  if (lasts == 0ull) return;                                             // (cannot be: the stretch holds mass)
  const bool over = hits == 0ull;                                        // rounding left the target at the very end: the last key with a weight
  const int from = over ? 63 - __clzll((long long)lasts) : __ffsll(hits) - 1;
  const int part = __shfl(over ? last : hit, from);
  before = __shfl(before, from);
  if (part % NW != wave) return;
  const int piece = part / NW;
  double sp = 0.0;
#pragma unroll
  for (int p = 0; p < K::P; ++p) sp = p == piece ? s[p] : sp;
  const double inc = wave_scan_d(sp);
  const unsigned long long lh = __ballot(!over && sp > 0.0 && before + inc > target), la = __ballot(sp > 0.0);
  const int at = lh ? __ffsll(lh) - 1 : 63 - __clzll((long long)la);
  if (lane != at) return;
  double c = before + (inc - sp);
  uint32_t kk = 0u;
  int pick = 0;
  bool done = false;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (e / K::VEC != piece || done) continue;
    const double w = kept(ks.key[e]);
    c += w;
    if (w > 0.0) {
      kk = ks.key[e];
      pick = ks.index(e);
      done = lh != 0ull && c > target;
    }
  }
  a.index[r] = pick;
  a.logp[r] = (float)(z_of(kk, kept.top, q.c2) - log_of(total));
}

// The thresholds of a row.  WALK(f) calls f(key) for all keys of the row, each by one thread of the workgroup.  WIDE: sums of masses over the row may pass
// 64 bits; a bin of the histogram is then two words, of the lower 39 bits (2^24 keys: 63 bits) and of the upper 6 of each weight
template <int NT, bool WIDE, typename WALK, typename S>
__device__ __forceinline__ uint32_t thresholds(const Draw& a, const Par& q, uint32_t top, uint32_t all, WALK walk, S& sh) {
  typedef std::conditional_t<WIDE, rr_u128, unsigned long long> M;
  constexpr int LIST = S::LISTED;
  M *red, *above_m;
  if constexpr (WIDE) { red = sh.redw; above_m = &sh.above_w; }
  else { red = sh.redm; above_m = &sh.above_m; }
  const int lane = threadIdx.x & 63;
  const double topd = (double)value_of(top);
  const float topv = value_of(top), per = (float)(22.180709777918249 * q.c2);      // 32 / T
  uint32_t cut = 1u;
  auto gather = [&](int bin, uint32_t from) {                            // the keys >= from of one bin into the list; how many they are
    __syncthreads();
    if (threadIdx.x == 0) sh.nlist = 0;
    __syncthreads();
    walk([&](uint32_t k) {
      if (k >= from && bin_of(k, topv, per) == bin) {
        const int at = atomicAdd(&sh.nlist, 1);
        if (at < LIST) sh.list[at] = k;
      }
    });
    __syncthreads();
    return sh.nlist;
  };
  auto each = [&](int n, int bin, uint32_t from, auto f) {               // f(key) for the bin's keys: from the list, or where they did not fit from the row
    if (n <= LIST) {
      for (int i = threadIdx.x; i < n; i += NT) f(sh.list[i]);
    } else {
      walk([&](uint32_t k) { if (k >= from && bin_of(k, topv, per) == bin) f(k); });
    }
  };
  auto ends = [&](int n, int bin, uint32_t from, uint32_t& lo, uint32_t& hi) {
    uint32_t h = 0u, l = 0u;                                             // l: of the complements
    each(n, bin, from, [&](uint32_t k) { h = k > h ? k : h; l = ~k > l ? ~k : l; });
    hi = block_max<NT>(h, sh.redu);
    lo = ~block_max<NT>(l, sh.redu);
  };
  if (q.k > 0 && all > (uint32_t)q.k) {
    for (int i = threadIdx.x; i < RR_DRAW_BINS; i += NT) sh.cnt[i] = 0u;
    __syncthreads();
    walk([&](uint32_t k) { if (k) atomicAdd(&sh.cnt[bin_of(k, topv, per)], 1u); });
    __syncthreads();
    find_bin<NT>([&](int b) { return sh.cnt[b]; }, (double)q.k, sh.redu, &sh.found, &sh.above_c);
    const int bin = sh.found;
    const uint32_t need = (uint32_t)q.k - sh.above_c;                    // the need-th largest of the bin
    const int n = gather(bin, 1u);
    if (n <= 256) {                                                      // the first wave alone, without barriers
      if (threadIdx.x < 64) {
        uint32_t k4[4], t = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) { k4[e] = lane + 64 * e < n ? sh.list[lane + 64 * e] : 0u; t = k4[e] > t ? k4[e] : t; }
        const uint32_t c = kth_largest(k4, (int)need, wave_max_u(t));
        if (lane == 0) sh.above_c = c;
      }
      __syncthreads();
      cut = sh.above_c;
    } else {
      uint32_t lo, hi;
      ends(n, bin, 1u, lo, hi);
      while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
        uint32_t c = 0u;
        each(n, bin, 1u, [&](uint32_t k) { c += k >= mid; });
        c = block_sum<NT>(c, sh.redu);
        if (c >= need) lo = mid; else hi = mid - 1u;
      }
      cut = lo;
    }
  }
  if (q.p > 0.0 && q.p < 1.0) {
    for (int i = threadIdx.x; i < RR_DRAW_BINS; i += NT) {
      sh.mass[i] = 0ull;
      if constexpr (WIDE) sh.cnt[i] = 0u;
    }
    __syncthreads();
    unsigned long long m = 0ull;                                         // (a thread's part of 2^24 keys: under 2^60)
    walk([&](uint32_t k) {
      if (k >= cut) {
        const unsigned long long w = steps_of(weight_of(k, top, topd, q.c2));
        m += w;
        if constexpr (WIDE) {
          const int b = bin_of(k, topv, per);
          if (w & 0x7fffffffffull) atomicAdd(&sh.mass[b], w & 0x7fffffffffull);
          if (w >> 39) atomicAdd(&sh.cnt[b], (uint32_t)(w >> 39));
        } else if (w) {
          atomicAdd(&sh.mass[bin_of(k, topv, per)], w);
        }
      }
    });
    const double lim = q.p * float_of(block_sum<NT>((M)m, red));         // (its barriers stand between the histogram's writes and reads)
    find_bin<NT>([&](int b) {
      if constexpr (WIDE) return ((rr_u128)sh.cnt[b] << 39) + sh.mass[b];
      else return sh.mass[b];
    }, lim, red, &sh.found, above_m);
    const int bin = sh.found;
    const double before = float_of(*above_m);
    const int n = gather(bin, cut);
    if (n <= 256) {
      if (threadIdx.x < 64) {
        uint32_t k4[4], t = 0u;
        unsigned long long w4[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          k4[e] = lane + 64 * e < n ? sh.list[lane + 64 * e] : 0u;
          w4[e] = k4[e] ? steps_of(weight_of(k4[e], top, topd, q.c2)) : 0ull;
          t = k4[e] > t ? k4[e] : t;
        }
        const uint32_t c = mass_threshold<4, unsigned long long>(k4, w4, wave_max_u(t), before, lim, sh.cnt, (unsigned long long*)sh.part, lane);
        if (lane == 0) sh.above_c = c;
      }
      __syncthreads();
      cut = sh.above_c;
    } else {
      uint32_t lo, hi;
      ends(n, bin, cut, lo, hi);
      while (lo < hi) {                                                  // the smallest value with less than lim strictly above it
        const uint32_t mid = lo + ((hi - lo) >> 1);
        unsigned long long s = 0ull;
        each(n, bin, cut, [&](uint32_t k) { if (k > mid) s += steps_of(weight_of(k, top, topd, q.c2)); });
        if (before + float_of(block_sum<NT>((M)s, red)) < lim) hi = mid; else lo = mid + 1u;
      }
      cut = lo;
    }
  }
  return cut;
}

// A row of any length by one workgroup.  ONE: the row's keys fit its registers; else stretch after stretch is loaded again for every walk.  WIDE: it may hold more than 2^18 keys
template <typename T, int NT, int E, bool ONE, bool WIDE, typename S>
__device__ __forceinline__ void draw_row(const Draw& a, int r, S& sh) {
  using K = Keys<T, NT, E>;
  const T* row = (const T*)a.logits + (long long)r * a.ld;
  const uint8_t* mask = a.mask ? a.mask + (long long)r * a.ldm : nullptr;
  const Par q = par_of(a, r);
  K ks;
  if constexpr (ONE) ks.load(row, mask, 0, a.V);
  auto walk_at = [&](auto f) {
    if constexpr (ONE) ks.each(f);
    else
      for (int b = 0; b < a.V; b += K::N) { ks.load(row, mask, b, a.V); ks.each(f); }
  };
  uint32_t top = 0u, n = 0u;
  walk_at([&](uint32_t k, int) { top = k > top ? k : top; n += k != 0u; });
  top = block_max<NT>(top, sh.redu);
  if (top == 0u) {
    if (threadIdx.x == 0) { a.index[r] = 0; a.logp[r] = -INFINITY; }
    return;
  }
  if (q.greedy) {
    uint32_t best = 0u;                                                  // ~index: the largest is the lowest index
    walk_at([&](uint32_t k, int i) { if (k == top && ~(uint32_t)i > best) best = ~(uint32_t)i; });
    best = block_max<NT>(best, sh.redu);
    if (threadIdx.x == 0) { a.index[r] = (int64_t)(~best); a.logp[r] = 0.f; }
    return;
  }
  if (q.k > 0 && q.k < a.V) n = block_sum<NT>(n, sh.redu);
  const uint32_t cut = thresholds<NT, WIDE>(a, q, top, n, [&](auto f) { walk_at([&](uint32_t k, int) { f(k); }); }, sh);
  const Kept kept = {top, cut, (double)value_of(top), q.c2, q.mp};
  if constexpr (ONE) {
    locate(a, q, r, ks, kept, 0.0, -1.0, sh);
  } else {
    double total = 0.0;
    auto stretch = [&](int b) {
      ks.load(row, mask, b, a.V);
      double s = 0.0;
      ks.each([&](uint32_t k, int) { s += kept(k); });
      return block_sum<NT>(s, sh.redd);
    };
    for (int b = 0; b < a.V; b += K::N) total += stretch(b);
    double before = 0.0, last_before = 0.0;
    int at = -1, last = 0;
    for (int b = 0; b < a.V && at < 0; b += K::N) {                      // (the same sums again: uniform)
      const double m = stretch(b);
      if (m > 0.0) { last = b; last_before = before; }
      if (before + m > q.u * total) at = b;
      else before += m;
    }
    if (at < 0) { at = last; before = last_before; }
    ks.load(row, mask, at, a.V);
    locate(a, q, r, ks, kept, before, total, sh);
  }
}
template <typename T, int NT, int E, bool ONE>
__global__ __launch_bounds__(NT) void k_draw_row(Draw a) {
  __shared__ Scratch<NT, 1024> sh;
  draw_row<T, NT, E, ONE, false>(a, blockIdx.x, sh);
}

// ---- few long rows: every stretch of a row has its own workgroup, five launches
//   top      the stretches' maxima and counts
//   measure  a histogram of the row (counts; masses too where top-p filters the whole row), or without a filter the stretches' masses
//   border   a workgroup a row: the bin of the border
//   gather   where all keys up to that bin are few, they go to a list with their indices, else the bin's keys do and the stretches' masses above it
//            are summed
//   pick     a workgroup a row: the thresholds among the list, the choice
// A row whose list would overflow is done by `pick` alone, walking all of it.  (Letting the last workgroup of a row go on instead of a launch took
// ten times as long: the fences that make the others' data visible across the eight L2s write them back.)
struct Long {
  uint32_t *tops, *counts;             // [R][C]
  double* masses;                      // [R][C]
  unsigned long long* mass;            // [R][bins] the lower 52 bits of the stretches' masses (at most 2^59 each, 1 024 of them) ...
  uint32_t* high;                      // [R][bins] ... and what is above
  uint32_t* cnt;                       // [R][bins]
  uint32_t *list, *where;              // [R][RR_DRAW_LIST]
  double *whole, *above;               // [R] the row's mass in steps, that above the border's bin
  uint32_t *top, *n;                   // [R]
  int *nlist, *mode, *bin, *greedy;      // [R]
  int C;
};
enum { RR_NOTHING = 0, RR_LIST_ALL = 1, RR_LIST_BORDER = 2, RR_ALONE = 3, RR_UNFILTERED = 4, RR_GREEDY = 5 };
struct LongScratch : Scratch<RR_DRAW_NT, RR_DRAW_LIST> {
  uint32_t where[RR_DRAW_LIST];
  rr_u128 redw[RR_DRAW_NT / 64], above_w;
};

__device__ __forceinline__ bool by_count(const Par& q, uint32_t n) { return q.k > 0 && n > (uint32_t)q.k; }
__device__ __forceinline__ bool by_mass(const Par& q) { return q.p > 0.0 && q.p < 1.0; }

template <typename T>
using LongKeys = Keys<T, RR_DRAW_NT, RR_DRAW_STRETCH / RR_DRAW_NT>;
template <typename T>
__device__ __forceinline__ void load_stretch(LongKeys<T>& ks, const Draw& a, int r, int c) {
  ks.load((const T*)a.logits + (long long)r * a.ld, a.mask ? a.mask + (long long)r * a.ldm : nullptr, c * RR_DRAW_STRETCH, a.V);
}
template <typename T>
__global__ __launch_bounds__(RR_DRAW_NT) void k_draw_top(Draw a, Long l) {
  __shared__ uint32_t red[RR_DRAW_NT / 64];
  const int r = blockIdx.x / l.C, c = blockIdx.x % l.C;
  LongKeys<T> ks;
  load_stretch<T>(ks, a, r, c);
  uint32_t top = 0u, n = 0u;
  ks.each([&](uint32_t k, int) { top = k > top ? k : top; n += k != 0u; });
  top = block_max<RR_DRAW_NT>(top, red);
  n = block_sum<RR_DRAW_NT>(n, red);
  if (threadIdx.x == 0) { l.tops[(long long)r * l.C + c] = top; l.counts[(long long)r * l.C + c] = n; }
  if (c == 0) {
    l.cnt[(long long)r * RR_DRAW_BINS + threadIdx.x] = 0u;
    l.mass[(long long)r * RR_DRAW_BINS + threadIdx.x] = 0ull;
    l.high[(long long)r * RR_DRAW_BINS + threadIdx.x] = 0u;
    if (threadIdx.x == 0) { l.nlist[r] = 0; l.greedy[r] = 0x7fffffff; }
  }
}

template <typename T>
__global__ __launch_bounds__(RR_DRAW_NT) void k_draw_measure(Draw a, Long l) {
  __shared__ LongScratch sh;
  constexpr int NT = RR_DRAW_NT;
  const int r = blockIdx.x / l.C, c = blockIdx.x % l.C, lane = threadIdx.x & 63;
  LongKeys<T> ks;
  load_stretch<T>(ks, a, r, c);
  const Par q = par_of(a, r);
  uint32_t top = 0u, n = 0u;                                             // the row's maximum and its number of keys, by each wave itself
  for (int i = lane; i < l.C; i += 64) {
    const uint32_t x = l.tops[(long long)r * l.C + i];
    top = x > top ? x : top;
    n += l.counts[(long long)r * l.C + i];
  }
  top = wave_max_u(top);
  n = wave_total(n);
  const bool counts = by_count(q, n), masses = !counts && by_mass(q);
  const int simple = top == 0u ? RR_NOTHING : q.greedy ? RR_GREEDY : !counts && !masses ? RR_UNFILTERED : -1;
  if (c == 0 && threadIdx.x == 0) { l.top[r] = top; l.n[r] = n; if (simple >= 0) l.mode[r] = simple; }
  if (top == 0u) return;
  if (q.greedy) {
    uint32_t best = 0u;
    ks.each([&](uint32_t k, int i) { if (k == top && ~(uint32_t)i > best) best = ~(uint32_t)i; });
    best = block_max<NT>(best, sh.redu);
    if (threadIdx.x == 0 && best) atomicMin(&l.greedy[r], (int)~best);
    return;
  }
  const double topd = (double)value_of(top);
  const float topv = value_of(top), per = (float)(22.180709777918249 * q.c2);
  if (simple == RR_UNFILTERED) {
    const Kept kept = {top, 1u, topd, q.c2, q.mp};
    double s = 0.0;
    ks.each([&](uint32_t k, int) { s += kept(k); });
    s = block_sum<NT>(s, sh.redd);
    if (threadIdx.x == 0) l.masses[(long long)r * l.C + c] = s;
    return;
  }
  sh.cnt[threadIdx.x] = 0u;
  sh.mass[threadIdx.x] = 0ull;
  __syncthreads();
  ks.each([&](uint32_t k, int) {
    if (k) {
      const int b = bin_of(k, topv, per);
      atomicAdd(&sh.cnt[b], 1u);
      if (masses) {
        const unsigned long long w = steps_of(weight_of(k, top, topd, q.c2));
        if (w) atomicAdd(&sh.mass[b], w);
      }
    }
  });
  __syncthreads();
  const long long at = (long long)r * RR_DRAW_BINS + threadIdx.x;
  if (sh.cnt[threadIdx.x]) atomicAdd(&l.cnt[at], sh.cnt[threadIdx.x]);
  const unsigned long long m = sh.mass[threadIdx.x];
  if (m) atomicAdd(&l.mass[at], m & 0xfffffffffffffull);
  if (m >> 52) atomicAdd(&l.high[at], (uint32_t)(m >> 52));
}

// a workgroup a row: the bin of the border, and how the row goes on
__global__ __launch_bounds__(RR_DRAW_NT) void k_draw_border(Draw a, Long l) {
  __shared__ uint32_t cnt[RR_DRAW_BINS], redu[RR_DRAW_NT / 64], above_c;
  __shared__ rr_u128 redw[RR_DRAW_NT / 64], above_w;
  __shared__ int found;
  constexpr int NT = RR_DRAW_NT;
  const int r = blockIdx.x;
  const uint32_t n = l.n[r];
  const Par q = par_of(a, r);
  if (l.top[r] == 0u || q.greedy || (!by_count(q, n) && !by_mass(q))) return;
  const bool counts = by_count(q, n), masses = !counts;
  const long long at = (long long)r * RR_DRAW_BINS + threadIdx.x;
  const uint32_t mine = l.cnt[at];
  const rr_u128 mym = ((rr_u128)l.high[at] << 52) + l.mass[at];
  cnt[threadIdx.x] = mine;
  if (threadIdx.x == 0) above_w = 0;
  const double whole = float_of(block_sum<NT>(mym, redw));
  if (counts) find_bin<NT>([&](int) { return mine; }, (double)q.k, redu, &found, &above_c);      // (a thread's own bin)
  else find_bin<NT>([&](int) { return mym; }, q.p * whole, redw, &found, &above_w);
  const int bin = found;
  const uint32_t upto = block_sum<NT>((int)threadIdx.x <= bin ? mine : 0u, redu), within = cnt[bin];
  if (threadIdx.x == 0) {
    l.mode[r] = upto <= RR_DRAW_LIST ? RR_LIST_ALL : masses && within <= RR_DRAW_LIST ? RR_LIST_BORDER : RR_ALONE;
    l.bin[r] = bin;
    l.whole[r] = whole;
    l.above[r] = float_of(above_w);
  }
}

// the row's choice among stretches with the masses `m(c)`: the stretch, the mass before it, the total
template <typename F>
__device__ __forceinline__ void pick_stretch(int C, double u, F m, int& at, double& before, double& total) {
  total = 0.0;
  for (int c = 0; c < C; ++c) total += m(c);
  double run = 0.0, last_before = 0.0;
  int last = 0;
  at = -1;
  for (int c = 0; c < C; ++c) {
    const double x = m(c);
    if (x > 0.0) { last = c; last_before = run; }
    if (at < 0 && run + x > u * total) { at = c; before = run; }
    run += x;
  }
  if (at < 0) { at = last; before = last_before; }
}

// a list in index order (a bitonic sort of sh.where, sh.list with it); `size`: the power of two >= 64 that holds it
__device__ __forceinline__ void sort_list(LongScratch& sh, int size) {
  for (int b = 2; b <= size; b <<= 1)
    for (int d = b >> 1; d > 0; d >>= 1) {
      __syncthreads();
      if ((int)threadIdx.x < size / 2) {
        const int i = ((int)threadIdx.x / d) * 2 * d + (int)threadIdx.x % d, j = i + d;
        const uint32_t pi = sh.where[i], pj = sh.where[j];
        if ((pi > pj) == ((i & b) == 0)) {
          sh.where[i] = pj; sh.where[j] = pi;
          const uint32_t t = sh.list[i];
          sh.list[i] = sh.list[j]; sh.list[j] = t;
        }
      }
    }
  __syncthreads();
}

// a workgroup a row: the thresholds among the list, the choice
template <typename T>
__global__ __launch_bounds__(RR_DRAW_NT) void k_draw_pick(Draw a, Long l) {
  __shared__ LongScratch sh;
  constexpr int NT = RR_DRAW_NT;
  const int r = blockIdx.x, mode = l.mode[r];
  const uint32_t top = l.top[r];
  const Par q = par_of(a, r);
  if (mode == RR_NOTHING || mode == RR_GREEDY) {
    if (threadIdx.x == 0) { a.index[r] = mode == RR_NOTHING ? 0 : l.greedy[r]; a.logp[r] = mode == RR_NOTHING ? -INFINITY : 0.f; }
    return;
  }
  if (mode == RR_ALONE) {
    draw_row<T, NT, RR_DRAW_STRETCH / NT, false, true>(a, r, sh);
    return;
  }
  const double topd = (double)value_of(top);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const bool counted = by_count(q, l.n[r]);
  if (mode == RR_UNFILTERED) {
    const Kept kept = {top, 1u, topd, q.c2, q.mp};
    int at;
    double before, total;
    pick_stretch(l.C, q.u, [&](int i) { return l.masses[(long long)r * l.C + i]; }, at, before, total);
    LongKeys<T> ks;
    load_stretch<T>(ks, a, r, at);
    locate(a, q, r, ks, kept, before, total, sh);
    return;
  }
  const int cnt = l.nlist[r];                                            // <= RR_DRAW_LIST = 2 NT
  const uint32_t* list = l.list + (long long)r * RR_DRAW_LIST;
  const uint32_t* where = l.where + (long long)r * RR_DRAW_LIST;
  uint32_t key[2], pos[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int i = threadIdx.x + NT * e;
    key[e] = i < cnt ? list[i] : 0u;
    pos[e] = i < cnt ? where[i] : 0xffffffffu;
  }
  const double whole = counted ? -1.0 : l.whole[r];              // what top-p refers to, in steps
  int size = 64;
  while (size < cnt) size <<= 1;                                         // <= RR_DRAW_LIST
  if (mode == RR_LIST_ALL && cnt <= 256) {                               // the first wave, as a short row
    __syncthreads();
    if (wave < 4) { sh.list[threadIdx.x] = key[0]; sh.where[threadIdx.x] = pos[0]; }
    sort_list(sh, size);
    if (wave > 0) return;
    uint32_t k4[4], p4[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) { k4[e] = sh.list[lane + 64 * e]; p4[e] = sh.where[lane + 64 * e]; }
    if (counted) {
      const uint32_t cut = kth_largest(k4, q.k, top);
#pragma unroll
      for (int e = 0; e < 4; ++e) k4[e] = k4[e] >= cut ? k4[e] : 0u;
      const int n = count_ge(k4, 1u);
      if (n <= 64) {
        wave_lds();
        int base = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const unsigned long long b = __ballot(k4[e] != 0u);
          const int at = base + __popcll(b & ((1ull << lane) - 1ull));
          if (k4[e]) { sh.list[at] = k4[e]; sh.where[at] = p4[e]; }
          base += __popcll(b);
        }
        wave_lds();
        uint32_t k1[1] = {lane < n ? sh.list[lane] : 0u};
        const int i1 = lane < n ? (int)sh.where[lane] : 0;
        choose<1>(a, q, r, k1, [&](int) { return i1; }, top, -1.0, nullptr, nullptr, lane);
        return;
      }
    }
    choose<4>(a, q, r, k4, [&](int e) { return (int)p4[e]; }, top, whole < 0.0 ? -1.0 : whole / RR_DRAW_STEP, sh.cnt, sh.part, lane);
    return;
  }
  auto extremes = [&](uint32_t& lo, uint32_t& hi) {
    uint32_t h = 0u, c = 0u;
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (key[e]) { h = key[e] > h ? key[e] : h; c = ~key[e] > c ? ~key[e] : c; }
    hi = block_max<NT>(h, sh.redu);
    lo = ~block_max<NT>(c, sh.redu);
  };
  uint32_t lo, hi;
  if (counted) {                                                         // the list holds everything from the border's bin on
    extremes(lo, hi);
    for (int step = 0; lo < hi; ++step) {
      const uint32_t mid = between(lo, hi, step) + 1u;
      const int c = (int)block_sum<NT>((uint32_t)((key[0] >= mid) + (key[1] >= mid)), sh.redu);
      if (c >= q.k) lo = mid; else hi = mid - 1u;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) key[e] = key[e] >= lo ? key[e] : 0u;
  }
  unsigned long long w[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) w[e] = key[e] ? steps_of(weight_of(key[e], top, topd, q.c2)) : 0ull;
  uint32_t cut = 1u;
  if (by_mass(q)) {
    const double m = counted ? (double)block_sum<NT>(w[0] + w[1], sh.redm) : whole;
    const double before = mode == RR_LIST_BORDER ? l.above[r] : 0.0;
    const double lim = q.p * m;
    extremes(lo, hi);
    for (int step = 0; lo < hi; ++step) {
      const uint32_t mid = between(lo, hi, step);
      const double s = before + (double)block_sum<NT>((key[0] > mid ? w[0] : 0ull) + (key[1] > mid ? w[1] : 0ull), sh.redm);
      if (s < lim) hi = mid; else lo = mid + 1u;
    }
    cut = lo;
  }
  const Kept kept = {top, cut, topd, q.c2, q.mp};
  if (mode == RR_LIST_BORDER) {                                          // a stretch's mass: its part above the bin and what the list has of it (whole steps: no order)
    const int C = l.C;
    int at;
    double before, total;
    __syncthreads();
    sh.mass[threadIdx.x] = 0ull;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (key[e] >= cut && kept(key[e]) > 0.0) atomicAdd(&sh.mass[pos[e] / RR_DRAW_STRETCH], w[e]);
    __syncthreads();
    pick_stretch(C, q.u, [&](int c) { return l.masses[(long long)r * C + c] + (double)sh.mass[c] / RR_DRAW_STEP; }, at, before, total);
    LongKeys<T> ks;
    load_stretch<T>(ks, a, r, at);
    locate(a, q, r, ks, kept, before, total, sh);
    return;
  }
  // everything is in the list: into index order, then as one stretch, two neighbours a thread
  __syncthreads();
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    sh.list[threadIdx.x + NT * e] = key[e];
    sh.where[threadIdx.x + NT * e] = pos[e];
  }
  sort_list(sh, size);
  double c[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) c[e] = 2 * (int)threadIdx.x + e < cnt ? kept(sh.list[2 * threadIdx.x + e]) : 0.0;
  const double inc = wave_scan_d(c[0] + c[1]);
  if (lane == 63) sh.redd[wave] = inc;
  if (threadIdx.x == 0) { sh.found = 0x7fffffff; sh.nlist = -1; }
  __syncthreads();
  double total = 0.0, base = 0.0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) { base = i == wave ? total : base; total += sh.redd[i]; }
  const double target = q.u * total, b0 = base + (inc - c[0] - c[1]);
  int hit = 0x7fffffff;
  if (c[0] > 0.0 && b0 + c[0] > target) hit = 2 * threadIdx.x;
  else if (c[1] > 0.0 && b0 + c[0] + c[1] > target) hit = 2 * threadIdx.x + 1;
  if (hit != 0x7fffffff) atomicMin(&sh.found, hit);
  if (c[0] > 0.0 || c[1] > 0.0) atomicMax(&sh.nlist, 2 * (int)threadIdx.x + (c[1] > 0.0 ? 1 : 0));
  __syncthreads();
  if (threadIdx.x == 0) {
    const int i = sh.found != 0x7fffffff ? sh.found : sh.nlist;          // (rounding may leave the target at the very end: the last key with a weight)
    a.index[r] = (int64_t)sh.where[i];
    a.logp[r] = (float)(z_of(sh.list[i], top, q.c2) - log_of(total));
  }
}

template <typename T>
__global__ __launch_bounds__(RR_DRAW_NT) void k_draw_gather(Draw a, Long l) {
  __shared__ uint32_t list[RR_DRAW_LIST], where[RR_DRAW_LIST];
  __shared__ double red[RR_DRAW_NT / 64];
  __shared__ int nlist, at_global;
  constexpr int NT = RR_DRAW_NT;
  const int r = blockIdx.x / l.C, c = blockIdx.x % l.C, mode = l.mode[r];
  if (mode != RR_LIST_ALL && mode != RR_LIST_BORDER) return;
  LongKeys<T> ks;
  load_stretch<T>(ks, a, r, c);
  const uint32_t top = l.top[r];
  const int bin = l.bin[r];
  const Par q = par_of(a, r);
  const float topv = value_of(top), per = (float)(22.180709777918249 * q.c2);
  if (threadIdx.x == 0) nlist = 0;
  __syncthreads();
  double s = 0.0;
  const Kept kept = {top, 1u, (double)topv, q.c2, q.mp};
  ks.each([&](uint32_t k, int i) {
    if (!k) return;
    const int b = bin_of(k, topv, per);
    if (b > bin) return;
    if (mode == RR_LIST_ALL || b == bin) {
      const int to = atomicAdd(&nlist, 1);                               // (at most the row's number, which fits)
      list[to] = k;
      where[to] = (uint32_t)i;
    } else s += kept(k);
  });
  __syncthreads();
  const int got = nlist;
  if (threadIdx.x == 0 && got) at_global = atomicAdd(&l.nlist[r], got);
  __syncthreads();
  for (int i = threadIdx.x; i < got; i += NT) {
    l.list[(long long)r * RR_DRAW_LIST + at_global + i] = list[i];
    l.where[(long long)r * RR_DRAW_LIST + at_global + i] = where[i];
  }
  if (mode == RR_LIST_BORDER) {
    s = block_sum<NT>(s, red);
    if (threadIdx.x == 0) l.masses[(long long)r * l.C + c] = s;
  }
}

// ------------------------------------------------------------------------------------------------ host
// rows that do not fit one workgroup's registers go by stretches, a workgroup each (4 096 x 131 072 float32, top-k and top-p: 1 580 us, 2 710 with a workgroup a row; 64 x 131 072:
// 45 and 133); a workgroup a row is quicker only where the rows just fill the chip and are hardly longer (256 x 20 000: 46 us against 55)
bool by_stretches(long long R, int V) { return V > 16384 && !(R >= 128 && R <= 512 && V <= 32768); }
int stretches(int V) { return (V + RR_DRAW_STRETCH - 1) / RR_DRAW_STRETCH; }
// rows of one pass over the five launches: what the workspace holds (33 KB a row up to 131 072 keys), and fewer than 2^32 threads
int rows_at_once(int V) {
  const int most = (1 << 21) / stretches(V);
  return most < 4096 ? most : 4096;
}
size_t long_bytes(long long R, int V) {
  const size_t C = (size_t)stretches(V);
  R = R < rows_at_once(V) ? R : rows_at_once(V);
  return (size_t)R * (C * 8 + RR_DRAW_BINS * 8 + 16 + C * 8 + RR_DRAW_BINS * 8 + RR_DRAW_LIST * 8 + 24);
}

template <typename T>
int draw_long(const Draw& a, void* ws, hipStream_t st) {
  Long l;
  const size_t R = (size_t)a.R, C = (size_t)stretches(a.V);
  char* p = (char*)ws;
  auto take = [&](size_t bytes) { void* at = p; p += bytes; return at; };
  l.masses = (double*)take(R * C * 8);
  l.mass = (unsigned long long*)take(R * RR_DRAW_BINS * 8);
  l.whole = (double*)take(R * 8);
  l.above = (double*)take(R * 8);
  l.tops = (uint32_t*)take(R * C * 4);
  l.counts = (uint32_t*)take(R * C * 4);
  l.high = (uint32_t*)take(R * RR_DRAW_BINS * 4);
  l.cnt = (uint32_t*)take(R * RR_DRAW_BINS * 4);
  l.list = (uint32_t*)take(R * RR_DRAW_LIST * 4);
  l.where = (uint32_t*)take(R * RR_DRAW_LIST * 4);
  l.nlist = (int*)take(R * 4);
  l.mode = (int*)take(R * 4);
  l.bin = (int*)take(R * 4);
  l.greedy = (int*)take(R * 4);
  l.top = (uint32_t*)take(R * 4);
  l.n = (uint32_t*)take(R * 4);
  l.C = (int)C;
  const dim3 grid((unsigned)(R * C)), one((unsigned)R), nt(RR_DRAW_NT);
  hipLaunchKernelGGL((k_draw_top<T>), grid, nt, 0, st, a, l);
  hipLaunchKernelGGL((k_draw_measure<T>), grid, nt, 0, st, a, l);
  hipLaunchKernelGGL(k_draw_border, one, nt, 0, st, a, l);
  hipLaunchKernelGGL((k_draw_gather<T>), grid, nt, 0, st, a, l);
  hipLaunchKernelGGL((k_draw_pick<T>), one, nt, 0, st, a, l);
  return rr_check(hipGetLastError());
}

template <typename T>
int draw_rows(const Draw& a, hipStream_t st) {
  const dim3 grid((unsigned)a.R);
  // the fewest threads whose registers hold the row (8 .. 32 keys each; 1 024 threads of 32 spill); what fits none is walked in stretches
  if (a.V <= 2048) hipLaunchKernelGGL((k_draw_row<T, 256, 8, true>), grid, dim3(256), 0, st, a);
  else if (a.V <= 4096) hipLaunchKernelGGL((k_draw_row<T, 256, 16, true>), grid, dim3(256), 0, st, a);
  else if (a.V <= 8192) hipLaunchKernelGGL((k_draw_row<T, 256, 32, true>), grid, dim3(256), 0, st, a);
  else if (a.V <= 16384) hipLaunchKernelGGL((k_draw_row<T, 512, 32, true>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((k_draw_row<T, 1024, 16, false>), grid, dim3(1024), 0, st, a);
  return rr_check(hipGetLastError());
}

template <typename T>
int draw_go(const Draw& a, bool stretches, void* ws, hipStream_t st) {
  const dim3 wg((unsigned)((a.R + 3) / 4)), wg16((unsigned)((a.R + 15) / 16));
  // without top-k and top-p rows of up to 128 keys take 16 lanes: the scans, the logarithm and the choice are paid once for four rows
  // (51 200 x 100 float32: 27 us with a wave a row)
  if (a.V <= 128 && a.pk == nullptr && a.pp == nullptr && (a.k <= 0 || a.k >= a.V) && !(a.p > 0.0 && a.p < 1.0)) {
    constexpr int N = rr_vec_of<T>::N;
    const bool vec = a.V % N == 0;
    if (vec && a.V <= 16 * N) hipLaunchKernelGGL((k_draw_group<T, N, true>), wg16, dim3(256), 0, st, a);
    else if (vec) hipLaunchKernelGGL((k_draw_group<T, 8, true>), wg16, dim3(256), 0, st, a);
    else if (a.V <= 32) hipLaunchKernelGGL((k_draw_group<T, 2, false>), wg16, dim3(256), 0, st, a);
    else if (a.V <= 64) hipLaunchKernelGGL((k_draw_group<T, 4, false>), wg16, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_draw_group<T, 8, false>), wg16, dim3(256), 0, st, a);
    return rr_check(hipGetLastError());
  }
  // up to 1 024 keys a wave a row (16 registers of keys a lane; 4 096 x 1 024 float32: 14 us, 20 with top-k and top-p; a workgroup a row: 19 and 49)
  if (a.V <= 64) hipLaunchKernelGGL((k_draw_wave<T, 1>), wg, dim3(256), 0, st, a);
  else if (a.V <= 128) hipLaunchKernelGGL((k_draw_wave<T, 2>), wg, dim3(256), 0, st, a);
  else if (a.V <= 256) hipLaunchKernelGGL((k_draw_wave<T, 4>), wg, dim3(256), 0, st, a);
  else if (a.V <= 512) hipLaunchKernelGGL((k_draw_wave<T, 8>), wg, dim3(256), 0, st, a);
  else if (a.V <= 1024) hipLaunchKernelGGL((k_draw_wave<T, 16>), wg, dim3(256), 0, st, a);
  else {
    return stretches ? draw_long<T>(a, ws, st) : draw_rows<T>(a, st);
  }
  return rr_check(hipGetLastError());
}

}  // namespace

extern "C" long long rr_draw_workspace(int R, int V) { return R > 0 && V > 0 && by_stretches(R, V) ? (long long)long_bytes(R, V) : 0; }

extern "C" int rr_draw(int dtype, const void* logits, long long ld, const uint8_t* mask, long long ldm, const float* uniforms, int64_t* index, float* logp, int R, int V,
                       double temperature, int top_k, double top_p, double min_p, const float* row_temperature, const int* row_top_k, const float* row_top_p,
                       const float* row_min_p, void* workspace, long long workspace_bytes, hipStream_t st) {
  if (dtype < RR_F32 || dtype > RR_BF16 || R < 0 || V < 1 || V > (1 << 24) || logits == nullptr || uniforms == nullptr || index == nullptr || logp == nullptr || ld < 0 || ldm < 0) return RR_EINVAL;
  if ((row_temperature == nullptr && !(temperature >= 0.0 && temperature < 1e30)) || (row_top_p == nullptr && !(top_p >= 0.0 && top_p <= 1.0)) ||
      (row_min_p == nullptr && !(min_p >= 0.0 && min_p <= 1.0)) || (row_top_k == nullptr && top_k < 0))
    return RR_EINVAL;
  if (R == 0) return RR_OK;
  if (by_stretches(R, V) && (workspace == nullptr || (size_t)workspace_bytes < long_bytes(R, V) || !rr_aligned16(workspace))) return RR_EINVAL;
  const Draw a = {logits, mask, uniforms, index, logp, row_temperature, row_top_p, row_min_p, row_top_k, temperature, 1.44269504088896340736 / temperature, top_p, min_p, ld, ldm,
                  top_k, R, V};
  // a launch holds fewer than 2^32 threads: at most 64 a row up to 1 024 keys, at most 1 024 beyond
  const int most = by_stretches(R, V) ? rows_at_once(V) : V <= 1024 ? 1 << 25 : 1 << 21, size = dtype == RR_F32 ? 4 : 2;
  for (long long r = 0; r < R; r += most) {
    Draw b = a;
    b.R = (int)(R - r < most ? R - r : most);
    b.logits = (const char*)logits + r * ld * size;
    if (mask != nullptr) b.mask += r * ldm;
    b.u += r;
    b.index += r;
    b.logp += r;
    if (b.pt != nullptr) b.pt += r;
    if (b.pk != nullptr) b.pk += r;
    if (b.pp != nullptr) b.pp += r;
    if (b.pm != nullptr) b.pm += r;
    const int rc = dtype == RR_F32 ? draw_go<float>(b, by_stretches(R, V), workspace, st)
                   : dtype == RR_F16 ? draw_go<rr_f16>(b, by_stretches(R, V), workspace, st)
                                     : draw_go<rr_bf16>(b, by_stretches(R, V), workspace, st);
    if (rc != RR_OK) return rc;
  }
  return RR_OK;
}
