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
// only kept keys pay for their 64-bit exponential.  Longer rows: a workgroup a row that walks the row several times (it stays in
// the L2): a histogram over the distance from the maximum, then only the keys of the bin that holds the border are looked at.  The
// histogram's masses are 64-bit integers in steps of 2^-45 (atomics on integers: the order does not matter).
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
  double t, p, mp;
  long long ld, ldm;
  int k, R, V;
};

struct Par { double t, p, mp, u; int k; bool greedy; };
__device__ __forceinline__ Par par_of(const Draw& a, int r) {
  Par q;
  const double t = a.pt ? (double)a.pt[r] : a.t;
  q.greedy = !(t > 0.0);                                       // 0 (and whatever is no temperature): the largest logit
  q.t = t;
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
__device__ __forceinline__ double z_of(uint32_t k, uint32_t top, double t) { return k == top ? 0.0 : ((double)value_of(k) - (double)value_of(top)) / t; }

// ---- wave helpers
__device__ __forceinline__ uint32_t wave_max_u(uint32_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const uint32_t x = __shfl_xor(v, o); v = v > x ? v : x; }
  return v;
}
__device__ __forceinline__ uint32_t wave_min_u(uint32_t v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) { const uint32_t x = __shfl_xor(v, o); v = v < x ? v : x; }
  return v;
}
__device__ __forceinline__ double wave_sum_d(double v) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
  return v;
}
__device__ __forceinline__ double wave_scan_d(double v, int lane) {      // inclusive
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double x = __shfl_up(v, o);
    if (lane >= o) v += x;
  }
  return v;
}

template <int E>
__device__ __forceinline__ int count_ge(const uint32_t (&key)[E], uint32_t at) {
  int n = 0;
#pragma unroll
  for (int q = 0; q < E; ++q) n += __popcll(__ballot(key[q] >= at));
  return n;
}
// the k-th largest of the wave's keys (k <= their number), top = the largest
template <int E>
__device__ __forceinline__ uint32_t kth_largest(const uint32_t (&key)[E], int k, uint32_t top) {
  uint32_t low = top;
#pragma unroll
  for (int q = 0; q < E; ++q) low = key[q] && key[q] < low ? key[q] : low;
  low = wave_min_u(low);
  uint32_t lo = low, hi = top;                                           // count(>= lo) >= k always holds; hi: the answer is <= hi
  while (lo < hi) {                                                      // (uniform; at most 32 halvings)
    const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
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

// keys (0: none) of one row in index order: register-major, lane-minor; idx of a register's key.  Writes the choice.
template <int E, typename IDX>
__device__ __forceinline__ void choose(const Draw& a, const Par& q, int r, uint32_t (&key)[E], IDX idx, uint32_t top, int lane) {
  double w[E], z = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    w[e] = key[e] ? exp(z_of(key[e], top, q.t)) : 0.0;
    z += w[e];
  }
  if (q.p > 0.0 && q.p < 1.0) {
    const double lim = q.p * wave_sum_d(z);
    uint32_t low = top;
#pragma unroll
    for (int e = 0; e < E; ++e) low = key[e] && key[e] < low ? key[e] : low;
    uint32_t lo = wave_min_u(low), hi = top;                             // the smallest value with less than lim strictly above it: mass(> top) = 0
    while (lo < hi) {
      const uint32_t mid = lo + ((hi - lo) >> 1);
      double m = 0.0;
      int n = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) m += key[e] > mid ? w[e] : 0.0;
      if (wave_sum_d(m) < lim) hi = mid; else lo = mid + 1u;
      // no key left between the two ends but one value: the next key from lo on is the threshold
#pragma unroll
      for (int e = 0; e < E; ++e) n += __popcll(__ballot(key[e] >= lo && key[e] <= hi));
      if (n <= 1) break;
    }
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
  double part[E], total = 0.0;                                           // a register's mass, in index order
  if constexpr (E == 1) {
    part[0] = total = wave_sum_d(w[0]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) { part[e] = wave_sum_d(w[e]); total += part[e]; }
  }
  const double target = q.u * total;
  // the register that the target falls in, then the lane; rounding may leave the target at the very end: the last key with a weight
  double before = 0.0, base = 0.0, we = 0.0;
  int reg = -1, last = -1;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (part[e] > 0.0) last = e;
    if (reg < 0 && before + part[e] > target) { reg = e; base = before; }
    before += part[e];
  }
  const bool over = reg < 0;
  if (over) reg = last;
  uint32_t ke = 0u;
  int ie = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e == reg) { we = w[e]; ke = key[e]; ie = idx(e); }
  const double cum = base + wave_scan_d(we, lane);
  const unsigned long long hit = __ballot(!over && we > 0.0 && cum > target), any = __ballot(we > 0.0);
  const int at = hit ? __ffsll((unsigned long long)hit) - 1 : 63 - __clzll((long long)any);
  if (lane == at) {
    a.index[r] = ie;
    a.logp[r] = (float)(z_of(ke, top, q.t) - log(total));
  }
}

template <typename T, int E>
__global__ __launch_bounds__(256) void k_draw_wave(Draw a) {
  __shared__ uint32_t skey[E > 1 ? 4 : 1][64];
  __shared__ int sidx[E > 1 ? 4 : 1][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.x * 4 + wave;
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
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        uint32_t k1[1] = {lane < n ? skey[wave][lane] : 0u};
        const int i1 = lane < n ? sidx[wave][lane] : 0;
        choose<1>(a, q, r, k1, [&](int) { return i1; }, top, lane);
        return;
      }
    }
  }
  choose<E>(a, q, r, key, [&](int e) { return lane + 64 * e; }, top, lane);
}

// ------------------------------------------------------------------------------------------------ long rows
#define RR_DRAW_BINS 1024
#define RR_DRAW_LIST 4096
#define RR_DRAW_STEP 35184372088832.0          // 2^45 steps a unit of weight

// bin of a key: its distance from the maximum in steps of T / 32 (monotone in the key), the last bin open
__device__ __forceinline__ int bin_of(uint32_t k, float topv, float per) {
  const float d = (topv - value_of(k)) * per;
  return d < (float)(RR_DRAW_BINS - 1) ? (int)d : (k && value_of(k) == topv ? 0 : RR_DRAW_BINS - 1);
}
__device__ __forceinline__ unsigned long long steps_of(double w) { return (unsigned long long)__double2ll_rn(w * RR_DRAW_STEP); }

template <typename T, int NT, bool VECTOR>
struct Row {
  static constexpr int VEC = VECTOR ? rr_vec_of<T>::N : 1, NW = NT / 64, PIECE = 64 * VEC;
  const T* row;
  const uint8_t* mask;
  int V, lane, wave, per_wave;                                           // pieces of a wave's stretch of the row
  __device__ __forceinline__ Row(const Draw& a, int r) {
    row = (const T*)a.logits + (long long)r * a.ld;
    mask = a.mask ? a.mask + (long long)r * a.ldm : nullptr;
    V = a.V; lane = threadIdx.x & 63; wave = threadIdx.x >> 6;
    per_wave = ((V + PIECE - 1) / PIECE + NW - 1) / NW;
  }
  __device__ __forceinline__ void load(int i0, uint32_t (&key)[VEC]) const {
    float x[VEC];
    if (i0 + VEC <= V) {
      rr_load_n<T, VEC>(row + i0, x);
      uint8_t m[VEC];
#pragma unroll
      for (int i = 0; i < VEC; ++i) m[i] = 1;
      if (mask != nullptr) __builtin_memcpy(m, mask + i0, VEC);
#pragma unroll
      for (int i = 0; i < VEC; ++i) key[i] = key_of(x[i], m[i] != 0);
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i) key[i] = i0 + i < V ? key_of((float)row[i0 + i], mask == nullptr || mask[i0 + i] != 0) : 0u;
    }
  }
  template <typename F>
  __device__ __forceinline__ void walk(F f) const {                      // f(key, index) for this lane's keys of its wave's stretch, in index order
    for (int p = wave * per_wave; p < (wave + 1) * per_wave && p * PIECE < V; ++p) {
      uint32_t key[VEC];
      const int i0 = p * PIECE + lane * VEC;
      load(i0, key);
#pragma unroll
      for (int i = 0; i < VEC; ++i) f(key[i], i0 + i);
    }
  }
};

template <int NT, typename V>
__device__ __forceinline__ V block_sum(V v, V* red) {                    // every thread gets the sum, added in a fixed order
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
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

// the first bin, from the top, at which the running sum of h reaches `need` (>= for counts, and for masses where need > 0): its number and the
// sum before it.  RR_DRAW_BINS where it is never reached.
template <int NT, typename V, typename R>
__device__ __forceinline__ void find_bin(const V* h, double need, R* red, int* found, V* above) {
  constexpr int PER = RR_DRAW_BINS / NT > 0 ? RR_DRAW_BINS / NT : 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = threadIdx.x * PER;
  V mine = 0;
  for (int i = 0; i < PER; ++i) mine += b0 + i < RR_DRAW_BINS ? h[b0 + i] : 0;
  V run = mine;                                                          // inclusive over the wave
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V x = __shfl_up(run, o);
    if (lane >= o) run += x;
  }
  __syncthreads();
  if (lane == 63) red[wave] = run;
  if (threadIdx.x == 0) *found = RR_DRAW_BINS;
  __syncthreads();
  V base = run - mine;
  for (int i = 0; i < wave; ++i) base += red[i];
  for (int i = 0; i < PER && b0 + i < RR_DRAW_BINS; ++i) {
    const V next = base + h[b0 + i];
    if ((double)base < need && (double)next >= need) { *found = b0 + i; *above = base; }      // one thread at the most: sums do not fall
    base = next;
  }
  __syncthreads();
}

template <typename T, int NT, bool VECTOR>
__global__ __launch_bounds__(NT) void k_draw_row(Draw a) {
  using Rw = Row<T, NT, VECTOR>;
  constexpr int NW = NT / 64;
  __shared__ unsigned long long mass[RR_DRAW_BINS];
  __shared__ uint32_t cnt[RR_DRAW_BINS];
  __shared__ uint32_t list[RR_DRAW_LIST];
  __shared__ double redd[NW];
  __shared__ unsigned long long redm[NW];
  __shared__ uint32_t redu[NW];
  __shared__ int found, nlist;
  __shared__ unsigned long long above_m;
  __shared__ uint32_t above_c;
  const int r = blockIdx.x;
  const Rw row(a, r);
  const Par q = par_of(a, r);
  uint32_t top = 0u;
  int ntop = 0;
  row.walk([&](uint32_t k, int) { top = k > top ? k : top; ntop += k != 0u; });
  top = block_max<NT>(top, redu);
  if (top == 0u) {
    if (threadIdx.x == 0) { a.index[r] = 0; a.logp[r] = -INFINITY; }
    return;
  }
  if (q.greedy) {
    uint32_t best = 0u;                                                  // ~index: the largest is the lowest index
    row.walk([&](uint32_t k, int i) { if (k == top && ~(uint32_t)i > best) best = ~(uint32_t)i; });
    best = block_max<NT>(best, redu);
    if (threadIdx.x == 0) { a.index[r] = (int64_t)(~best); a.logp[r] = 0.f; }
    return;
  }
  const float topv = value_of(top), per = (float)(32.0 / q.t);
  uint32_t cut = 1u;                                                     // keys from here on are kept
  // gathers the keys >= from of one bin into `list`, the thresholds are then found among them; false where they do not fit
  auto gather = [&](int bin, uint32_t from) {
    __syncthreads();
    if (threadIdx.x == 0) nlist = 0;
    __syncthreads();
    row.walk([&](uint32_t k, int) {
      if (k >= from && k && bin_of(k, topv, per) == bin) {
        const int at = atomicAdd(&nlist, 1);
        if (at < RR_DRAW_LIST) list[at] = k;
      }
    });
    __syncthreads();
    return nlist;
  };
  auto each = [&](int n, int bin, uint32_t from, auto f) {               // f(key) for the bin's keys: from the list, or where they did not fit from the row
    if (n <= RR_DRAW_LIST) {
      for (int i = threadIdx.x; i < n; i += NT) f(list[i]);
    } else {
      row.walk([&](uint32_t k, int) { if (k >= from && k && bin_of(k, topv, per) == bin) f(k); });
    }
  };
  auto ends = [&](int n, int bin, uint32_t from, uint32_t& lo, uint32_t& hi) {
    uint32_t h = 0u, l = 0u;                                             // l: of the complements
    each(n, bin, from, [&](uint32_t k) { h = k > h ? k : h; l = ~k > l ? ~k : l; });
    hi = block_max<NT>(h, redu);
    lo = ~block_max<NT>(l, redu);
  };
  if (q.k > 0 && q.k < a.V) {
    const uint32_t all = (uint32_t)block_sum<NT>((uint32_t)ntop, redu);
    if (all > (uint32_t)q.k) {
      for (int i = threadIdx.x; i < RR_DRAW_BINS; i += NT) cnt[i] = 0u;
      __syncthreads();
      row.walk([&](uint32_t k, int) { if (k) atomicAdd(&cnt[bin_of(k, topv, per)], 1u); });
      __syncthreads();
      find_bin<NT>(cnt, (double)q.k, redu, &found, &above_c);
      const int bin = found;
      const uint32_t need = (uint32_t)q.k - above_c;                     // the need-th largest of the bin
      const int n = gather(bin, 1u);
      uint32_t lo, hi;
      ends(n, bin, 1u, lo, hi);
      while (lo < hi) {
        const uint32_t mid = lo + ((hi - lo) >> 1) + 1u;
        uint32_t c = 0u;
        each(n, bin, 1u, [&](uint32_t k) { c += k >= mid; });
        c = block_sum<NT>(c, redu);
        if (c >= need) lo = mid; else hi = mid - 1u;
      }
      cut = lo;
    }
  }
  if (q.p > 0.0 && q.p < 1.0) {
    for (int i = threadIdx.x; i < RR_DRAW_BINS; i += NT) mass[i] = 0ull;
    __syncthreads();
    unsigned long long m = 0ull;
    row.walk([&](uint32_t k, int) {
      if (k >= cut) {
        const unsigned long long w = steps_of(exp(z_of(k, top, q.t)));
        m += w;
        if (w) atomicAdd(&mass[bin_of(k, topv, per)], w);
      }
    });
    m = block_sum<NT>(m, redm);                                          // (its barriers stand between the histogram's writes and reads)
    const double lim = q.p * (double)m;
    find_bin<NT>(mass, lim, redm, &found, &above_m);
    const int bin = found;
    const unsigned long long before = above_m;
    const int n = gather(bin, cut);
    uint32_t lo, hi;
    ends(n, bin, cut, lo, hi);
    while (lo < hi) {                                                    // the smallest value with less than lim strictly above it
      const uint32_t mid = lo + ((hi - lo) >> 1);
      unsigned long long s = 0ull;
      each(n, bin, cut, [&](uint32_t k) { if (k > mid) s += steps_of(exp(z_of(k, top, q.t))); });
      s = before + block_sum<NT>(s, redm);
      if ((double)s < lim) hi = mid; else lo = mid + 1u;
    }
    cut = lo;
  }
  // masses of the waves' stretches, in index order; then the stretch that holds the target, split over all threads
  auto weight = [&](uint32_t k) {
    if (k < cut || k == 0u) return 0.0;
    const double w = exp(z_of(k, top, q.t));
    return q.mp > 0.0 && w < q.mp ? 0.0 : w;
  };
  double s = 0.0;
  row.walk([&](uint32_t k, int) { s += weight(k); });
  s = wave_sum_d(s);
  __syncthreads();
  if (row.lane == 0) redd[row.wave] = s;
  __syncthreads();
  double total = 0.0, base = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) total += redd[i];
  const double target = q.u * total;
  int seg = -1, last = 0;
  double run = 0.0;
#pragma unroll
  for (int i = 0; i < NW; ++i) {
    if (redd[i] > 0.0) last = i;
    if (seg < 0 && run + redd[i] > target) { seg = i; base = run; }
    run += redd[i];
  }
  if (seg < 0) { seg = last; base = run - redd[last]; }
  // consecutive keys of the stretch to consecutive threads, `per_t` each
  const int first = seg * row.per_wave * Rw::PIECE, len = row.per_wave * Rw::PIECE, per_t = (len + NT - 1) / NT;
  const int i0 = first + threadIdx.x * per_t;
  const int end = first + len < a.V ? first + len : a.V;
  auto at = [&](int i) { return key_of((float)row.row[i], row.mask == nullptr || row.mask[i] != 0); };
  s = 0.0;
  for (int i = i0; i < i0 + per_t && i < end; ++i) s += weight(at(i));
  double inc = wave_scan_d(s, row.lane);
  __syncthreads();
  if (row.lane == 63) redd[row.wave] = inc;
  if (threadIdx.x == 0) { found = 0x7fffffff; nlist = -1; }
  __syncthreads();
  for (int i = 0; i < row.wave; ++i) base += redd[i];
  double c = base + inc - s;
  int pick = 0x7fffffff, lastp = -1;
  for (int i = i0; i < i0 + per_t && i < end; ++i) {
    const double w = weight(at(i));
    c += w;
    if (w > 0.0) {
      lastp = i;
      if (c > target) { pick = i; break; }
    }
  }
  if (pick != 0x7fffffff) atomicMin(&found, pick);
  if (lastp >= 0) atomicMax(&nlist, lastp);
  __syncthreads();
  if (threadIdx.x == 0) {
    const int i = found != 0x7fffffff ? found : nlist;                   // (rounding may leave the target at the very end: the last key with a weight)
    a.index[r] = i;
    a.logp[r] = (float)(z_of(at(i), top, q.t) - log(total));
  }
}

template <typename T>
int draw_go(const Draw& a, hipStream_t st) {
  const dim3 wg((unsigned)((a.R + 3) / 4));
  // a wave a row up to 1 024 keys (16 registers of keys a lane); beyond that 256 threads a row, 1 024 where a row is long enough to feed them
  if (a.V <= 64) hipLaunchKernelGGL((k_draw_wave<T, 1>), wg, dim3(256), 0, st, a);
  else if (a.V <= 128) hipLaunchKernelGGL((k_draw_wave<T, 2>), wg, dim3(256), 0, st, a);
  else if (a.V <= 256) hipLaunchKernelGGL((k_draw_wave<T, 4>), wg, dim3(256), 0, st, a);
  else if (a.V <= 512) hipLaunchKernelGGL((k_draw_wave<T, 8>), wg, dim3(256), 0, st, a);
  else if (a.V <= 1024) hipLaunchKernelGGL((k_draw_wave<T, 16>), wg, dim3(256), 0, st, a);
  else {
    const int e = 16 / (int)sizeof(T);
    const bool vec = a.ld % e == 0 && rr_aligned16(a.logits);
    if (a.V <= 8192) {
      if (vec) hipLaunchKernelGGL((k_draw_row<T, 256, true>), dim3((unsigned)a.R), dim3(256), 0, st, a);
      else hipLaunchKernelGGL((k_draw_row<T, 256, false>), dim3((unsigned)a.R), dim3(256), 0, st, a);
    } else {
      if (vec) hipLaunchKernelGGL((k_draw_row<T, 1024, true>), dim3((unsigned)a.R), dim3(1024), 0, st, a);
      else hipLaunchKernelGGL((k_draw_row<T, 1024, false>), dim3((unsigned)a.R), dim3(1024), 0, st, a);
    }
  }
  return rr_check(hipGetLastError());
}

}  // namespace

extern "C" int rr_draw(int dtype, const void* logits, long long ld, const uint8_t* mask, long long ldm, const float* uniforms, int64_t* index, float* logp, int R, int V,
                       double temperature, int top_k, double top_p, double min_p, const float* row_temperature, const int* row_top_k, const float* row_top_p,
                       const float* row_min_p, hipStream_t st) {
  if (R < 0 || V < 1 || V > (1 << 24) || logits == nullptr || uniforms == nullptr || index == nullptr || logp == nullptr || ld < 0 || ldm < 0) return RR_EINVAL;
  if ((row_temperature == nullptr && !(temperature >= 0.0 && temperature < 1e30)) || (row_top_p == nullptr && !(top_p >= 0.0 && top_p <= 1.0)) ||
      (row_min_p == nullptr && !(min_p >= 0.0 && min_p <= 1.0)) || (row_top_k == nullptr && top_k < 0))
    return RR_EINVAL;
  if (R == 0) return RR_OK;
  const Draw a = {logits, mask, uniforms, index, logp, row_temperature, row_top_p, row_min_p, row_top_k, temperature, top_p, min_p, ld, ldm, top_k, R, V};
  switch (dtype) {
    case RR_F32: return draw_go<float>(a, st);
    case RR_F16: return draw_go<rr_f16>(a, st);
    case RR_BF16: return draw_go<rr_bf16>(a, st);
  }
  return RR_EINVAL;
}
