// Sampling codes from logits: temperature, top-k, top-p and min-p, one given random number per row.
//
// MATHEMATICS.  Order the row's codes by (logit descending, index ascending); e_i = exp((z_i - max z) / T).  All three cuts keep a
// prefix of that order (top-k: its first k; top-p: every code with less than p of the kept mass before it; min-p: e_i >= min_p), so the
// kept set is {z > t} and the first r codes, by index, of those with z == t.  t and r are found by counts for top-k and by mass for
// top-p, in bins: of the row first (linear in z), then of the codes of the one bin that the cut falls into; nothing is sorted.  The code
// is the lowest kept index at which the running kept mass passes u times its total.
//
// NUMBERS.  e is computed in 64 bits (good to 2^-44 of itself) and held as a whole number of 2^(down - 61) in 64 bits, and all sums are of
// whole numbers: atomics in any order give the same bits, and so do the forms below.  `down` lets a row's sum fit 62 bits.  Up to 512 codes it is
// log2 V rounded up, less 1; beyond, it goes by the row's own sum, estimated first: a row of one large logit keeps nearly all the bits for the far
// ones.  (One unit for all rows of a length, 2^-38 at 2^24 codes, lost a tail of 2^-15 of the row whole.)  A cut and a draw fall on the side that
// exact arithmetic gives them unless p or u lies within 2^-44 + V 2^-53 (V <= 512) or 2^-44 + 2.25 V 2^-61 of a border, 2^-39 at 2^20 codes and
// 2^-35 at 2^24; a sum in fp64, one code after the other, is good to V 2^-53.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "group_kernel.hpp"   // GroupNum: conversions of the row types

namespace qinco {

struct SampleArgs {
  const void* logits;   // (n, V), rows `stride` elements apart
  long stride;
  long n;
  int V;
  const void* u;        // (n), fp32 or fp64
  int u_f64;
  // per-row arrays, or null and the scalar next to them
  const float* T_rows;
  double T;
  const int* k_rows;
  int k;
  const float* p_rows;
  double p;
  const float* m_rows;
  double m;
  void* codes;
  int codes_i64;
  float* logp;          // nullable
  int down;             // V <= 512: of every row (SampleMass)
};

// the row's settings, with every switched-off cut in the form that keeps everything
struct SampleRow {
  double y, p, m, u;   // y: log2(e) / T
  int k;
  bool greedy;
};

// 1 / x for x > 0: the hardware's estimate and two Newton steps, good to the last bit or two (a tiny or infinite x: the estimate alone)
__device__ __forceinline__ double sample_reciprocal(double x) {
  const double e = __builtin_amdgcn_rcp(x);
  double r = fma(fma(-x, e, 1.0), e, e);
  r = fma(fma(-x, r, 1.0), r, r);
  return r == r ? r : e;
}

__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, long r) {
  SampleRow s;
  const double T = a.T_rows ? (double)a.T_rows[r] : a.T;
  s.greedy = !(T > 0.0);
  s.y = s.greedy ? 1.0 : 1.4426950408889634074 * sample_reciprocal(T);
  // (T = inf: every finite logit has the same mass; 1 / T = inf: nothing but the largest has any.  0 * inf and inf - inf stay out of it)
  s.y = fmin(fmax(s.y, 1e-290), 1e290);
  s.k = a.k_rows ? a.k_rows[r] : a.k;
  if (s.k <= 0 || s.k > a.V) s.k = a.V;
  s.p = a.p_rows ? (double)a.p_rows[r] : a.p;
  if (!(s.p < 1.0)) s.p = 1.0;
  if (s.p < 0.0) s.p = 0.0;
  s.m = a.m_rows ? (double)a.m_rows[r] : a.m;
  if (!(s.m > 0.0)) s.m = 0.0;
  if (s.m > 1.0) s.m = 1.0;
  const double u = a.u_f64 ? reinterpret_cast<const double*>(a.u)[r] : (double)reinterpret_cast<const float*>(a.u)[r];
  s.u = u > 0.0 ? (u < 1.0 ? u : 1.0) : 0.0;
  return s;
}

__device__ __forceinline__ void sample_answer(const SampleArgs& a, long r, long code, float logp) {
  if (a.codes_i64) reinterpret_cast<long long*>(a.codes)[r] = code;
  else reinterpret_cast<int*>(a.codes)[r] = (int)code;
  if (a.logp) a.logp[r] = logp;
}

// a logit as the kernels hold it: NaN is -inf (never drawn), as is everything behind the row's end
template <typename T>
__device__ __forceinline__ float sample_logit(const T* z, int i, int V) {
  const float x = i < V ? GroupNum<T>::get(z[i]) : -INFINITY;
  return x == x ? x : -INFINITY;
}
// fp32 -> unsigned, order-preserving; -0 counts as +0
__device__ __forceinline__ unsigned sample_key(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float sample_unkey(unsigned k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }
constexpr unsigned kSampleKeyMasked = 0x007FFFFFu;   // sample_key(-inf)

// the row's own constants
struct SampleMass {
  struct Power { double b; int k; };   // 2^k b
  double zmax, y, least;
  int down;
  double c[12];   // of 2^f: (ln 2)^n / n!
  // top: max z.  An infinite one stands as a number above all others: what equals it has an argument above 0, everything else one far below
  __device__ __forceinline__ SampleMass(float top, double log2e_T, int down_) : zmax(top < INFINITY ? (double)top : 1.7e308), y(log2e_T) {
    scale(down_);
    constexpr double l = 0.69314718055994530942;
    c[0] = 1.0;
    c[1] = l;
#pragma unroll
    for (int n = 2; n < 12; ++n) c[n] = c[n - 1] * l / n;
    // (kept in scalar registers: as literals the compiler moves each into a vector register pair again before every product)
#pragma unroll
    for (int n = 1; n < 12; ++n) asm("" : "+s"(c[n]));
  }
  // masses as whole numbers of 2^(down_ - 61); at 2^least one is zero: least rounds to down_ - 61, a quarter below it
  __device__ __forceinline__ void scale(int down_) {
    down = down_;
    least = (double)(down_ - 61) - 0.25;
  }
  // log2 of e = exp((z - max z) / T)
  __device__ __forceinline__ double arg(float z) const { return fmin(fmax(((double)z - zmax) * y, least), 0.0); }
  // 2^x for -62 < x <= 0: x = k + f with |f| <= 1/2 (the sum with 1.5 2^52 rounds x to k and leaves it in the low word), b = the series of
  // exp(f ln 2) to the 11th power (what is left out is below (ln 2 / 2)^12 / 12! = 7e-15)
  __device__ __forceinline__ Power power(float z) const {
    const double x = arg(z), k = x + 0x1.8p52, f = x - (k - 0x1.8p52);
    double b = c[11];
#pragma unroll
    for (int n = 10; n >= 0; --n) b = fma(b, f, c[n]);
    return Power{b, __double2loint(k)};
  }
  static __device__ __forceinline__ double value(Power e) { return __hiloint2double(__double2hiint(e.b) + (e.k << 20), __double2loint(e.b)); }
  // b < 1.42 in 52 bits (the sum with 2^52 rounds it to 2^-51), the sum's exponent shifted out, then down to the unit: at least 2, at most 63
  // places, what falls off is dropped
  __device__ __forceinline__ unsigned long long whole(Power e) const {
    return ((unsigned long long)__double_as_longlong(fma(e.b, 0x1p51, 0x1p52)) << 12) >> (2 + down - e.k);
  }
  __device__ __forceinline__ unsigned long long q(float z) const { return whole(power(z)); }
  __device__ __forceinline__ unsigned long long q(float z, double m) const {   // ... zero for what min-p cuts
    const Power e = power(z);
    return value(e) >= m ? whole(e) : 0ull;
  }
  // natural logarithm of a code's share of `total` (1 <= total 2^(down - 61) < 2^25): that is 2^k b with 2/3 < b <= 4/3, and
  // log b = 2 (s + s^3 / 3 + s^5 / 5 + ...), s = (b - 1) / (b + 1), |s| <= 1/5, to s^19 (what is left out is below 1e-15)
  __device__ __forceinline__ float logp(float z, unsigned long long total) const {
    const double v = (double)total;
    int k = (__double2hiint(v) >> 20) - 1023;
    double b = __hiloint2double((__double2hiint(v) & 0xFFFFF) | 1023 << 20, __double2loint(v));
    if (b > 4.0 / 3.0) {
      b *= 0.5;
      ++k;
    }
    k -= 61 - down;
    const double s = (b - 1.0) * sample_reciprocal(b + 1.0), s2 = s * s;
    double p = 1.0 / 19.0;
    p = fma(p, s2, 1.0 / 17.0);
    p = fma(p, s2, 1.0 / 15.0);
    p = fma(p, s2, 1.0 / 13.0);
    p = fma(p, s2, 1.0 / 11.0);
    p = fma(p, s2, 1.0 / 9.0);
    p = fma(p, s2, 1.0 / 7.0);
    p = fma(p, s2, 1.0 / 5.0);
    p = fma(p, s2, 1.0 / 3.0);
    p = fma(p * s2, s, s);
    return (float)fma(0.69314718055994530942, arg(z) - (double)k, -2.0 * p);
  }
};

// A logit that no code of mass is at or below: 62 powers of two under the largest one, and one fp32 further down.  A top-k that reaches codes
// without mass changes nothing, so they are not counted, nor sought in their bin (which most of a row can share).
__device__ __forceinline__ float sample_massless(float zmax, double y) {
  const double z = (zmax < INFINITY ? (double)zmax : 1.7e308) - 62.0 * sample_reciprocal(y);
  return sample_unkey(sample_key((float)fmax(z, -3.40282346638528859812e38)) - 1);   // (below the lowest fp32: -inf)
}

// smallest whole number that is at least p * total (and at least 1): "mass before < p * total" is "mass before < this"
__device__ __forceinline__ unsigned long long sample_bound(double p, unsigned long long total) {
  const unsigned long long v = (unsigned long long)ceil(p * (double)total);
  return v < 1 ? 1 : (v > total ? total : v);
}
// mass that the draw falls on: the first code whose running mass is above it
__device__ __forceinline__ unsigned long long sample_target(double u, unsigned long long total) {
  const unsigned long long v = (unsigned long long)(u * (double)total);
  return v < total ? v : total - 1;
}
// smallest r with r q >= rem, at most 2^25 (the quotient in 64 bits is off by less than one)
__device__ __forceinline__ unsigned sample_ceil_div(unsigned long long rem, unsigned long long q) {
  if (rem <= q) return rem ? 1 : 0;
  unsigned r = (unsigned)fmin(ceil((double)rem / (double)q), 0x1p25);
  if ((r - 1) * q >= rem) --r;
  if (r * q < rem) ++r;
  return r;
}

// Wave-wide sums and scans by DPP (rows of 16 lanes shifted, then broadcast over the rows behind): every lane has to be active.
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned sample_dpp(unsigned v) {   // 0 where the step has no source lane
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long sample_dpp(unsigned long long v) {
  return (unsigned long long)sample_dpp<CTRL, ROWS>((unsigned)(v >> 32)) << 32 | sample_dpp<CTRL, ROWS>((unsigned)v);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ float sample_dpp(float v) { return __uint_as_float(sample_dpp<CTRL, ROWS>(__float_as_uint(v))); }
template <typename T>
__device__ __forceinline__ T sample_wave_scan(T v) {   // inclusive
  v += sample_dpp<0x111, 0xf>(v);
  v += sample_dpp<0x112, 0xf>(v);
  v += sample_dpp<0x114, 0xf>(v);
  v += sample_dpp<0x118, 0xf>(v);
  v += sample_dpp<0x142, 0xa>(v);
  v += sample_dpp<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ unsigned sample_lane(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ unsigned long long sample_lane(unsigned long long v, int lane) {
  return (unsigned long long)sample_lane((unsigned)(v >> 32), lane) << 32 | sample_lane((unsigned)v, lane);
}
__device__ __forceinline__ float sample_lane(float v, int lane) { return __uint_as_float(sample_lane(__float_as_uint(v), lane)); }
template <typename T>
__device__ __forceinline__ T sample_wave_sum(T v) { return sample_lane(sample_wave_scan(v), 63); }
__device__ __forceinline__ unsigned sample_wave_max(unsigned v) {
  v = max(v, sample_dpp<0x111, 0xf>(v));
  v = max(v, sample_dpp<0x112, 0xf>(v));
  v = max(v, sample_dpp<0x114, 0xf>(v));
  v = max(v, sample_dpp<0x118, 0xf>(v));
  v = max(v, sample_dpp<0x142, 0xa>(v));
  v = max(v, sample_dpp<0x143, 0xc>(v));
  return sample_lane(v, 63);
}
// what the wave's lanes wrote to LDS is there for its other lanes (the LDS executes a wave's accesses in order: nothing to wait for)
__device__ __forceinline__ void sample_wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Bins of the first look at a row, linear in z: 0 holds the largest logit, the last one the smallest, or whatever lies 62 or more powers
// of two below it (no mass).  fp32 subtraction and product are monotone and a NaN (both infinite) goes to the last bin with everything
// that can be below it, so a bin never holds a logit above one of an earlier bin.
struct SampleBins {
  float zmax, c, last;
  __device__ __forceinline__ int of(float z) const { return (int)fminf((zmax - z) * c, last); }
};
__device__ __forceinline__ SampleBins sample_bins(float zmax, float zmin, double y, int bins) {
  const float range = fminf((zmax - zmin) * (float)y, 62.f);   // (any c > 0 will do: its rounding moves bins, not codes)
  const float c = range > 0.f ? fminf((float)bins * (float)y * __builtin_amdgcn_rcpf(range), 3e38f) : 0.f;
  return SampleBins{zmax, zmax < INFINITY ? c : 0.f, (float)(bins - 1)};
}

// ---------------------------------------------------------------------------------------------------------------------
// G = 16 or 32 lanes per row, V <= G R: the row stays in registers (lane l holds codes l R ... l R + R - 1), no barrier anywhere.  What is done
// once per row (scans, bounds, the logarithm) is two thirds of the instructions of a wave per row; here two or four rows share it.
// Both cuts look at 64 bins of the row first (counts and masses by LDS atomics, 64 / G bins per lane), then at the few codes of the one bin
// that the cut falls into.  A bin of more than 64 codes (heavy ties) is searched bit by bit instead.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSampleGroupThreads = 256;
struct SampleGroupLds {
  unsigned long long mass[64];
  unsigned long long m_mass[64];   // codes of the bin in question
  unsigned count[64];
  float m_z[64];
  float t;                         // what one lane found for all
  unsigned r;
  unsigned long long q;
};

// over the G lanes of a row (16: a DPP row; 32: two of them)
template <int G, typename T>
__device__ __forceinline__ T sample_row_scan(T v) {   // inclusive
  v += sample_dpp<0x111, 0xf>(v);
  v += sample_dpp<0x112, 0xf>(v);
  v += sample_dpp<0x114, 0xf>(v);
  v += sample_dpp<0x118, 0xf>(v);
  if (G == 32) v += sample_dpp<0x142, 0xa>(v);
  return v;
}
template <int G, typename T>
__device__ __forceinline__ T sample_row_last(T v) {   // the last lane's, in every lane
  return G == 16 ? sample_dpp<0x15F, 0xf>(v) : __shfl(v, 31, 32);
}
template <int G, typename T>
__device__ __forceinline__ T sample_row_sum(T v) {    // in every lane: by rotations
  v += sample_dpp<0x128, 0xf>(v);
  v += sample_dpp<0x124, 0xf>(v);
  v += sample_dpp<0x122, 0xf>(v);
  v += sample_dpp<0x121, 0xf>(v);
  if (G == 32) v += __shfl_xor(v, 16, 32);
  return v;
}
template <int G>
__device__ __forceinline__ unsigned sample_row_max(unsigned v) {
  v = max(v, sample_dpp<0x128, 0xf>(v));
  v = max(v, sample_dpp<0x124, 0xf>(v));
  v = max(v, sample_dpp<0x122, 0xf>(v));
  v = max(v, sample_dpp<0x121, 0xf>(v));
  if (G == 32) v = max(v, __shfl_xor(v, 16, 32));
  return v;
}

template <typename T, int G, int R>
__global__ void __launch_bounds__(kSampleGroupThreads) sample_group_kernel(SampleArgs a, long row0) {
  constexpr int ROWS = kSampleGroupThreads / G, PB = 64 / G;   // rows of a workgroup, bins of a lane
  __shared__ SampleGroupLds lds[ROWS];
  SampleGroupLds& s = lds[threadIdx.x / G];
  const int l = threadIdx.x % G, V = a.V, row_shift = (threadIdx.x & 63) / G * G;
  // lanes of this row among a ballot's
  auto mine = [&](unsigned long long ballot) { return (unsigned)(ballot >> row_shift) & (unsigned)((1ull << G) - 1); };
  // (a row's lanes take every branch together: the branches below may part rows, never a row)
  const long row = row0 + (long)blockIdx.x * ROWS + threadIdx.x / G;
  if (row >= a.n) return;
  const T* logits = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const SampleRow set = sample_row(a, row);
  float z[R];
  {
    constexpr int U = R * sizeof(T) < 16 ? R : 16 / sizeof(T);   // codes of one load
    struct alignas(sizeof(T)) Raw { T v[U]; };
#pragma unroll
    for (int j = 0; j < R; j += U) {
      const int i = l * R + j;
      if (i + U <= V) {
        const Raw raw = *reinterpret_cast<const Raw*>(logits + i);
#pragma unroll
        for (int e = 0; e < U; ++e) {
          const float x = GroupNum<T>::get(raw.v[e]);
          z[j + e] = x == x ? x : -INFINITY;
        }
      } else {
#pragma unroll
        for (int e = 0; e < U; ++e) z[j + e] = sample_logit(logits, i + e, V);
      }
    }
  }
  float hi = z[0], lo = INFINITY;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    hi = fmaxf(hi, z[j]);
    lo = fminf(lo, z[j] > -INFINITY ? z[j] : INFINITY);
  }
  const float zmax = sample_unkey(sample_row_max<G>(sample_key(hi)));
  if (zmax == -INFINITY) {
    if (l == 0) sample_answer(a, row, -1, -INFINITY);
    return;
  }
  if (set.greedy) {
    const int first = __builtin_ctz(mine(__ballot(hi == zmax)));
    int at = 0;
#pragma unroll
    for (int j = R - 1; j >= 0; --j) at = z[j] == zmax ? j : at;
    if (l == first) sample_answer(a, row, l * R + at, 0.f);
    return;
  }
  const SampleMass mass(zmax, set.y, a.down);
  unsigned long long q[R];
  unsigned floored = 0;   // bit j: cut by min-p
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const SampleMass::Power e = mass.power(z[j]);
    q[j] = mass.whole(e);
    floored |= (mass.value(e) >= set.m ? 0u : 1u) << j;
    if ((j & 1) == 1) __builtin_amdgcn_sched_barrier(0);   // (two exponentials at a time: more side by side only take registers)
  }
  float t = -INFINITY;
  unsigned r = 0;
  const bool by_count = set.k < V, by_mass = set.p < 1.0;
  if (by_count || by_mass) {
    const float zmin = sample_unkey(~sample_row_max<G>(~sample_key(lo)));
    const SampleBins bins = sample_bins(zmax, zmin, set.y, 64);
    const float massless = sample_massless(zmax, set.y);
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      s.mass[l * PB + j] = 0;
      s.count[l * PB + j] = 0;
    }
    sample_wave_sync();
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int b = bins.of(z[j]);
      if (z[j] > massless) atomicAdd(&s.count[b], 1u);
      if (q[j]) atomicAdd(&s.mass[b], q[j]);
    }
    sample_wave_sync();
    unsigned c_in[PB], c_sum = 0;
    unsigned long long m_in[PB], m_sum = 0;
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      c_sum += c_in[j] = s.count[l * PB + j];
      m_sum += m_in[j] = s.mass[l * PB + j];
    }
    const unsigned c_run = sample_row_scan<G>(c_sum), c_all = sample_row_last<G>(c_run);
    const unsigned long long m_run = sample_row_scan<G>(m_sum);
    unsigned long long total = sample_row_last<G>(m_run);   // mass of what top-k keeps
    // codes of bin b into m_z, m_mass; their number
    auto members = [&](int b) {
      unsigned in = 0;
#pragma unroll
      for (int j = 0; j < R; ++j) in |= (unsigned)(z[j] > massless && bins.of(z[j]) == b) << j;
      const unsigned n = __builtin_popcount(in), run = sample_row_scan<G>(n);
      unsigned to = run - n;
      if (in) {
#pragma unroll
        for (int j = 0; j < R; ++j) {
          if (in >> j & 1) {
            if (to < 64) {
              s.m_z[to] = z[j];
              s.m_mass[to] = q[j];
            }
            ++to;
          }
        }
      }
      sample_wave_sync();
      return (int)sample_row_last<G>(run);
    };
    int kb = 64, n_kb = 0;        // the bin that top-k cuts, 64: none; its codes
    unsigned long long qt = 0;    // mass of a code at t
    if (by_count && (unsigned)set.k < c_all) {
      unsigned want = (unsigned)set.k - (c_run - c_sum);
      unsigned long long above = m_run - m_sum;
      int b = l * PB;
#pragma unroll
      for (int j = 0; j < PB - 1; ++j) {
        const bool on = b == l * PB + j && want > c_in[j];
        want -= on ? c_in[j] : 0;
        above += on ? m_in[j] : 0;
        b += on;
      }
      const int src = __builtin_ctz(mine(__ballot(c_run >= (unsigned)set.k)));
      want = __shfl(want, src, G);
      above = __shfl(above, src, G);
      kb = __shfl(b, src, G);
      n_kb = members(kb);
      if (n_kb <= 64) {
        for (int i = l; i < n_kb; i += G) {
          const float mz = s.m_z[i];
          unsigned gt = 0, ge = 0;
          for (int o = 0; o < n_kb; ++o) {
            gt += s.m_z[o] > mz;
            ge += s.m_z[o] >= mz;
          }
          if (gt < want && want <= ge) {   // (equal logits find the same)
            s.t = mz;
            s.r = want - gt;
            s.q = s.m_mass[i];
          }
        }
        sample_wave_sync();
        t = s.t;
        r = s.r;
        qt = s.q;
        unsigned long long in = 0;
        if (by_mass)
          for (int i = l; i < n_kb; i += G) in += s.m_z[i] > t ? s.m_mass[i] : 0ull;
        total = above + sample_row_sum<G>(in) + r * qt;
      } else {   // the largest t that at least k codes reach, a bit at a time
        unsigned key = 0;
        for (int b = 31; b >= 0; --b) {
          const unsigned c = key | 1u << b;
          unsigned n = 0;
#pragma unroll
          for (int j = 0; j < R; ++j) n += sample_key(z[j]) >= c;
          if (sample_row_sum<G>(n) >= (unsigned)set.k) key = c;
        }
        t = sample_unkey(key);
        unsigned n = 0;
        unsigned long long m = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) {
          n += z[j] > t;
          m += z[j] > t ? q[j] : 0ull;
        }
        r = (unsigned)set.k - sample_row_sum<G>(n);
        qt = mass.q(t);
        total = sample_row_sum<G>(m) + r * qt;
      }
    }
    if (by_mass) {
      const unsigned long long bound = sample_bound(set.p, total);
      // (a bin that top-k cuts counts as reached: what it keeps of it is in `total`)
      unsigned long long need = bound - (m_run - m_sum);
      int b = l * PB;
#pragma unroll
      for (int j = 0; j < PB - 1; ++j) {
        const bool on = b == l * PB + j && need > m_in[j];
        need -= on ? m_in[j] : 0;
        b += on;
      }
      const int src = __builtin_ctz(mine(__ballot(m_run >= bound)));
      need = __shfl(need, src, G);
      const int pb = __shfl(b, src, G);
      const int n = pb == kb ? n_kb : members(pb);
      if (n <= 64) {
        s.r = 0;
        sample_wave_sync();
        unsigned long long in = 0;
        for (int i = l; i < n; i += G) {
          const float mz = s.m_z[i];
          if (mz > t) {
            const unsigned long long mq = s.m_mass[i];
            unsigned long long gt = 0, eq = 0;
            for (int o = 0; o < n; ++o) {
              const float x = s.m_z[o];
              const unsigned long long m = s.m_mass[o];
              gt += x > mz ? m : 0ull;
              eq += x == mz ? m : 0ull;
            }
            if (gt < need && need <= gt + eq) {
              s.t = mz;
              s.r = sample_ceil_div(need - gt, mq);
            }
            in += mq;
          }
        }
        sample_wave_sync();
        if (s.r) {
          t = s.t;
          r = s.r;
        } else {   // on the ties that top-k kept
          r = min(r, sample_ceil_div(need - sample_row_sum<G>(in), qt));
        }
      } else {
        const unsigned kt = sample_key(t);
        const unsigned long long at_t = r * qt;
        unsigned key = 0;
        for (int b = 31; b >= 0; --b) {
          const unsigned c = key | 1u << b;
          unsigned long long m = 0;
#pragma unroll
          for (int j = 0; j < R; ++j) m += sample_key(z[j]) >= c && z[j] > t ? q[j] : 0ull;
          if (sample_row_sum<G>(m) + (kt >= c ? at_t : 0ull) >= bound) key = c;
        }
        const float x = sample_unkey(key);
        unsigned long long m = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) m += z[j] > x && z[j] > t ? q[j] : 0ull;
        const unsigned rr = sample_ceil_div(bound - sample_row_sum<G>(m) - (kt > key ? at_t : 0ull), mass.q(x));
        r = key == kt ? min(r, rr) : rr;
        t = x;
      }
    }
  }
  // the draw: kept masses summed in index order
  unsigned nth = 0;
  if (r) {
    unsigned ties = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) ties += z[j] == t;
    nth = sample_row_scan<G>(ties) - ties;
  }
  unsigned long long sum = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const bool tie = z[j] == t;
    const bool kept = (z[j] > t || (tie && nth < r)) && !(floored >> j & 1);
    nth += tie;
    q[j] = kept ? q[j] : 0ull;
    sum += q[j];
  }
  const unsigned long long run = sample_row_scan<G>(sum), total = sample_row_last<G>(run);
  const unsigned long long target = sample_target(set.u, total);
  if (run > target && run - sum <= target) {
    unsigned long long upto = run - sum;
    int at = 0;
    float x = 0.f;
    bool found = false;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      upto += q[j];
      if (!found && upto > target) {
        found = true;
        at = j;
        x = z[j];
      }
    }
    sample_answer(a, row, l * R + at, mass.logp(x, total));
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// One wave per row, V <= 64 R: the row stays in registers (lane l holds codes l R ... l R + R - 1), no barrier anywhere.
// Both cuts look at 64 bins of the row first (counts and masses by LDS atomics, scanned by the wave), then at the few codes of the one
// bin that the cut falls into, a lane each.  A bin of more than 64 codes (heavy ties) is searched bit by bit instead.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSampleRowWaves = 4;
struct SampleWaveLds {
  unsigned long long mass[64];
  unsigned count[64];
  unsigned long long m_mass[64];   // codes of the bin in question
  float m_z[64];
};

template <int R>
struct SampleWaveRow {
  float z[R];
  unsigned long long q[R];

  // codes of bin b into m_z, m_mass; their number, or -1 if more than 64
  __device__ __forceinline__ int members(SampleWaveLds& s, const SampleBins& bins, int b) const {
    const int lane = threadIdx.x & 63;
    int n = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool in = q[j] && bins.of(z[j]) == b;
      const unsigned long long at = __ballot(in);
      const int to = n + (int)__builtin_popcountll(at & ((1ull << lane) - 1));
      if (in && to < 64) {
        s.m_z[to] = z[j];
        s.m_mass[to] = q[j];
      }
      n += (int)__builtin_popcountll(at);
    }
    return n <= 64 ? n : -1;
  }
};

// (Five waves per SIMD asked for: left alone the compiler takes 104 registers for 8 codes per lane instead of 88, 16384 x 512 42 us instead of 39.)
template <typename T, int R>
__global__ void __launch_bounds__(64 * kSampleRowWaves, 5) sample_wave_kernel(SampleArgs a, long row0) {
  __shared__ SampleWaveLds lds[kSampleRowWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // (known to be the same in every lane: the row's settings are scalars)
  SampleWaveLds& s = lds[wave];
  const int lane = threadIdx.x & 63, V = a.V;
  const long row = row0 + (long)blockIdx.x * kSampleRowWaves + wave;
  if (row >= a.n) return;
  const T* logits = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const SampleRow set = sample_row(a, row);
  SampleWaveRow<R> w;
  float hi = -INFINITY, lo = INFINITY;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    w.z[j] = sample_logit(logits, lane * R + j, V);
    hi = fmaxf(hi, w.z[j]);
    lo = fminf(lo, w.z[j] > -INFINITY ? w.z[j] : INFINITY);
  }
  const float zmax = sample_unkey(sample_wave_max(sample_key(hi)));
  if (zmax == -INFINITY) {
    if (lane == 0) sample_answer(a, row, -1, -INFINITY);
    return;
  }
  if (set.greedy) {
    const int first = __builtin_ctzll(__ballot(hi == zmax));
    int at = 0;
#pragma unroll
    for (int j = R - 1; j >= 0; --j) at = w.z[j] == zmax ? j : at;
    if (lane == first) sample_answer(a, row, lane * R + at, 0.f);
    return;
  }
  const SampleMass mass(zmax, set.y, a.down);
  unsigned floored = 0;   // bit j: cut by min-p
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const SampleMass::Power e = mass.power(w.z[j]);
    w.q[j] = mass.whole(e);
    floored |= (mass.value(e) >= set.m ? 0u : 1u) << j;
    if ((j & 3) == 3) __builtin_amdgcn_sched_barrier(0);   // (four exponentials at a time: more side by side only take registers)
  }
  float t = -INFINITY;
  unsigned r = 0;
  const bool by_count = set.k < V, by_mass = set.p < 1.0;
  if (by_count || by_mass) {
    const float zmin = sample_unkey(~sample_wave_max(~sample_key(lo)));
    const SampleBins bins = sample_bins(zmax, zmin, set.y, 64);
    s.mass[lane] = 0;
    s.count[lane] = 0;
    sample_wave_sync();
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (w.q[j]) {
        const int b = bins.of(w.z[j]);
        atomicAdd(&s.count[b], 1u);
        atomicAdd(&s.mass[b], w.q[j]);
      }
    }
    sample_wave_sync();
    const unsigned c_in = s.count[lane], c_run = sample_wave_scan(c_in);
    const unsigned long long m_in = s.mass[lane], m_run = sample_wave_scan(m_in);
    unsigned long long total = sample_lane(m_run, 63);   // mass of what top-k keeps
    int kb = 64;                                         // the bin that top-k cuts, 64: none
    int n_kb = 0;
    unsigned long long qt = 0;                           // mass of a code at t
    if (by_count && (unsigned)set.k < sample_lane(c_run, 63)) {
      kb = __builtin_ctzll(__ballot(c_run >= (unsigned)set.k));
      const unsigned want = (unsigned)set.k - (sample_lane(c_run, kb) - sample_lane(c_in, kb));
      const unsigned long long above = sample_lane(m_run, kb) - sample_lane(m_in, kb);
      n_kb = w.members(s, bins, kb);
      sample_wave_sync();
      if (n_kb >= 0) {
        const float mz = lane < n_kb ? s.m_z[lane] : -INFINITY;
        const unsigned long long mq = lane < n_kb ? s.m_mass[lane] : 0ull;
        unsigned gt = 0, ge = 0;
        for (int i = 0; i < n_kb; ++i) {
          const float o = __uint_as_float(sample_lane(__float_as_uint(mz), i));
          gt += o > mz;
          ge += o >= mz;
        }
        const int at = __builtin_ctzll(__ballot(lane < n_kb && gt < want && want <= ge));
        t = __uint_as_float(sample_lane(__float_as_uint(mz), at));
        r = want - sample_lane(gt, at);
        qt = sample_lane(mq, at);
        total = above + sample_wave_sum(mz > t ? mq : 0ull) + r * qt;
      } else {   // the largest t that at least k keys reach, a bit at a time
        unsigned key = 0;
        for (int b = 31; b >= 0; --b) {
          const unsigned c = key | 1u << b;
          unsigned n = 0;
#pragma unroll
          for (int j = 0; j < R; ++j) n += (unsigned)__builtin_popcountll(__ballot(sample_key(w.z[j]) >= c));
          if (n >= (unsigned)set.k) key = c;
        }
        t = sample_unkey(key);
        unsigned n = 0;
        unsigned long long m = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) {
          n += (unsigned)__builtin_popcountll(__ballot(w.z[j] > t));
          m += w.z[j] > t ? w.q[j] : 0ull;
        }
        r = (unsigned)set.k - n;
        qt = mass.q(t);
        total = sample_wave_sum(m) + r * qt;
      }
    }
    if (by_mass) {
      const unsigned long long bound = sample_bound(set.p, total);
      // (a bin that top-k cuts counts as reached: what it keeps of it is in `total`)
      const unsigned long long reach = __ballot(m_run >= bound);
      const int pb = min(reach ? __builtin_ctzll(reach) : 63, kb);
      const unsigned long long need = bound - (sample_lane(m_run, pb) - sample_lane(m_in, pb));
      const int n = pb == kb ? n_kb : w.members(s, bins, pb);
      sample_wave_sync();
      if (n >= 0) {
        const float mz = lane < n ? s.m_z[lane] : -INFINITY;
        unsigned long long mq = lane < n ? s.m_mass[lane] : 0ull;
        if (!(mz > t)) mq = 0;
        unsigned long long gt = 0, ge = 0;
        for (int i = 0; i < n; ++i) {
          const float o = __uint_as_float(sample_lane(__float_as_uint(mz), i));
          const unsigned long long m = sample_lane(mq, i);
          gt += o > mz ? m : 0ull;
          ge += o >= mz ? m : 0ull;
        }
        const unsigned long long hit = __ballot(mz > t && gt < need && need <= ge);
        if (hit) {   // (else it falls on the ties that top-k kept)
          const int at = __builtin_ctzll(hit);
          t = __uint_as_float(sample_lane(__float_as_uint(mz), at));
          r = sample_ceil_div(need - sample_lane(gt, at), sample_lane(mq, at));
        } else {
          r = min(r, sample_ceil_div(need - sample_wave_sum(mq), qt));
        }
      } else {
        const unsigned kt = sample_key(t);
        const unsigned long long at_t = r * qt;
        unsigned key = 0;
        for (int b = 31; b >= 0; --b) {
          const unsigned c = key | 1u << b;
          unsigned long long m = 0;
#pragma unroll
          for (int j = 0; j < R; ++j) m += sample_key(w.z[j]) >= c && w.z[j] > t ? w.q[j] : 0ull;
          if (sample_wave_sum(m) + (kt >= c ? at_t : 0ull) >= bound) key = c;
        }
        const float z = sample_unkey(key);
        unsigned long long m = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) m += w.z[j] > z && w.z[j] > t ? w.q[j] : 0ull;
        const unsigned rr = sample_ceil_div(bound - sample_wave_sum(m) - (kt > key ? at_t : 0ull), mass.q(z));
        r = key == kt ? min(r, rr) : rr;
        t = z;
      }
    }
  }
  // the draw: kept masses summed in index order
  unsigned ties = 0, nth = 0;
  if (r) {
#pragma unroll
    for (int j = 0; j < R; ++j) ties += w.z[j] == t;
    nth = sample_wave_scan(ties) - ties;
  }
  unsigned long long sum = 0;
#pragma unroll
  for (int j = 0; j < R; ++j) {
    const bool tie = w.z[j] == t;
    const bool kept = (w.z[j] > t || (tie && nth < r)) && !(floored >> j & 1);
    nth += tie;
    w.q[j] = kept ? w.q[j] : 0ull;
    sum += w.q[j];
  }
  const unsigned long long run = sample_wave_scan(sum), total = sample_lane(run, 63);
  const unsigned long long target = sample_target(set.u, total);
  const int first = __builtin_ctzll(__ballot(run > target));
  if (lane == first) {
    unsigned long long upto = run - sum;
    int at = 0;
    float z = 0.f;
    bool found = false;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      upto += w.q[j];
      if (!found && upto > target) {
        found = true;
        at = j;
        z = w.z[j];
      }
    }
    sample_answer(a, row, lane * R + at, mass.logp(z, total));
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Longer rows, by workgroups of NT threads and 1024 bins.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSampleBins = 1024;

template <int NT>
struct SampleBlock {   // scratch of the workgroup's scans
  unsigned long long m[NT / 64];
  unsigned c[NT / 64];
};
// Exclusive scan over the workgroup's threads of a mass and a count, and their totals; the value of the last one to need its shared
// memory is read before the barrier that ends it.
template <int NT>
__device__ __forceinline__ void sample_block_scan(SampleBlock<NT>& s, unsigned long long m, unsigned c, unsigned long long& m_before,
                                                  unsigned& c_before, unsigned long long& m_all, unsigned& c_all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const unsigned long long mi = sample_wave_scan(m);
  const unsigned ci = sample_wave_scan(c);
  if (lane == 63) {
    s.m[w] = mi;
    s.c[w] = ci;
  }
  __syncthreads();
  // the waves' sums: a lane each, scanned again
  const unsigned long long mw = lane < NT / 64 ? s.m[lane] : 0ull;
  const unsigned cw = lane < NT / 64 ? s.c[lane] : 0u;
  const unsigned long long ms = sample_wave_scan(mw);
  const unsigned cs = sample_wave_scan(cw);
  m_all = sample_lane(ms, NT / 64 - 1);
  c_all = sample_lane(cs, NT / 64 - 1);
  const int wu = __builtin_amdgcn_readfirstlane(w);
  m_before = sample_lane(ms, wu) - sample_lane(mw, wu) + mi - m;
  c_before = sample_lane(cs, wu) - sample_lane(cw, wu) + ci - c;
  __syncthreads();
}

struct SampleFound {   // what one thread found for all
  int bin;
  unsigned count;
  unsigned long long mass;
};

// The key at which a running sum over keys in descending order reaches `target` (1 <= target <= its total): bins of the range [lo, hi] that
// the key lies in, 10 bits at a time.  each(f) calls f(key, amount) for this thread's share of the codes; `before` = the sum above the key.
template <int NT, typename Each>
__device__ __forceinline__ unsigned sample_search(SampleBlock<NT>& blk, SampleFound& found, unsigned long long* bins, unsigned lo, unsigned hi,
                                                  unsigned long long target, unsigned long long& before, Each each) {
  constexpr int PB = kSampleBins / NT;
  before = 0;
  for (;;) {
    const unsigned span = hi - lo;
    const int shift = span < kSampleBins ? 0 : 22 - __builtin_clz(span);
    for (int b = threadIdx.x; b < kSampleBins; b += NT) bins[b] = 0;
    __syncthreads();
    each([&](unsigned key, auto amount) {
      if (key >= lo && key <= hi) {
        const unsigned long long v = amount();
        if (v) atomicAdd(&bins[(hi - key) >> shift], v);
      }
    });
    __syncthreads();
    unsigned long long m = 0, m_before, m_all;
    unsigned none, none_all;
#pragma unroll
    for (int j = 0; j < PB; ++j) m += bins[threadIdx.x * PB + j];
    sample_block_scan<NT>(blk, m, 0u, m_before, none, m_all, none_all);
    if (m_before < target && target <= m_before + m) {
#pragma unroll
      for (int j = 0; j < PB; ++j) {
        const unsigned long long n = bins[threadIdx.x * PB + j];
        if (m_before < target && target <= m_before + n) {
          found.bin = threadIdx.x * PB + j;
          found.mass = m_before;
        }
        m_before += n;
      }
    }
    __syncthreads();
    const unsigned b = (unsigned)found.bin;
    before += found.mass;
    target -= found.mass;
    hi -= b << shift;
    if (shift == 0) return hi;
    const unsigned width = (1u << shift) - 1;
    lo = hi - lo > width ? hi - width : lo;
  }
}

// The draw among N codes per thread, in the order of their threads, with `run` of mass and `seen` codes at t before the first thread's: codes
// above t, and those at t that are among the first r.  index(j) = the code that z[j] is the logit of.  Barriers inside: every thread.
template <int NT, int N, typename Index>
__device__ __forceinline__ void sample_draw(const SampleArgs& a, long row, const float (&z)[N], Index index, const SampleMass& mass, double m,
                                            float t, unsigned r, unsigned long long qt, SampleBlock<NT>& blk, unsigned long long run,
                                            unsigned seen, unsigned long long target, unsigned long long total) {
  unsigned long long q[N], sum = 0;
  unsigned at_t = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    q[j] = 0;
    if (z[j] > t) q[j] = mass.q(z[j], m);
    sum += q[j];
    at_t += z[j] == t && r > 0;
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
  }
  unsigned long long before, all;
  unsigned c_before, c_all;
  sample_block_scan<NT>(blk, sum, at_t, before, c_before, all, c_all);
  run += before + (min(seen + c_before, r) - min(seen, r)) * qt;
  seen += c_before;
  const unsigned long long here = sum + (min(seen + at_t, r) - min(seen, r)) * qt;
  if (run <= target && target < run + here) {
    int at = 0;
    float x = 0.f;
    bool drawn = false;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const bool tie = z[j] == t && r > 0;
      run += q[j] + (tie && seen < r ? qt : 0ull);
      seen += tie;
      if (!drawn && run > target) {
        drawn = true;
        at = index(j);
        x = z[j];
      }
    }
    sample_answer(a, row, at, mass.logp(x, total));
  }
}

// One workgroup per row, V <= NT R, the row and its masses in registers: thread t holds codes t steps ... t steps + steps - 1.  The codes of
// the bin that a cut falls into are listed, and up to 64 of them compared by one wave, a lane each; more (heavy ties) are searched in bins.
// One scan over the threads, of the mass above t and of the codes at t, gives the total and the thread that the draw falls on.  Every
// exponential is taken once (of what top-k keeps alone, where nothing else wants them) and kept: 8000 rows of 4099 fp16 go in 88 us without
// a cut, 110 with a top-k of 40 and 133 with all three, one row of 10240 in 15; with the row in LDS and the exponentials taken anew in each pass
// they took two thirds longer.  Bound by instructions: 86, 97 and 125 vector ones per 64 codes, issued 0.90, 0.79 and 0.85 of the time.  (Loads of
// 16 bytes for two-byte types, eight codes, are worth 1 us of the 88.)
template <typename T, int NT, int R>
__global__ void __launch_bounds__(NT, 4) sample_block_kernel(SampleArgs a, long row0) {
  constexpr int PB = kSampleBins / NT, PAIR = 2;
  static_assert(PB * NT == kSampleBins && R % 4 == 0 && R <= 32, "bins per thread, groups of a row, bits of a mask");
  __shared__ unsigned long long bin_mass[kSampleBins], part[kSampleBins];
  __shared__ unsigned bin_count[kSampleBins];
  __shared__ SampleBlock<NT> blk;
  __shared__ SampleFound found;
  __shared__ unsigned range[2][NT / 64], key_range[2], upper;
  __shared__ unsigned long long m_mass[64];
  __shared__ float m_z[64];
  __shared__ int n_listed[2];   // by top-k, by top-p
  __shared__ struct {
    float t;
    unsigned r;
    unsigned long long in;
  } cut;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.V;
  const int steps = (V + NT - 1) / NT, i0 = tid * steps;
  const long row = row0 + blockIdx.x;
  const T* logits = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const SampleRow set = sample_row(a, row);
  float z[R], hi = -INFINITY, lo = INFINITY;
#pragma unroll
  for (int j = 0; j < R; j += 4) {
    if (j + 4 <= steps && i0 + j + 4 <= V) {
      GroupUnit<T, 4> u;
      u.load(logits + i0 + j);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = GroupNum<T>::get(u.v[e]);
        z[j + e] = x == x ? x : -INFINITY;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[j + e] = j + e < steps ? sample_logit(logits, i0 + j + e, V) : -INFINITY;
    }
  }
#pragma unroll
  for (int j = 0; j < R; ++j) {
    hi = fmaxf(hi, z[j]);
    lo = fminf(lo, z[j] > -INFINITY ? z[j] : INFINITY);
  }
  // f(j, logit) for this thread's codes, two at a time.  (The logit in a form that what is made of it is not kept from one pass to the
  // next, nor taken out of a loop: a key or a bin is fewer instructions than a spilled register.)
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < R; j += PAIR) {
      if (j < steps) {
#pragma unroll
        for (int e = 0; e < PAIR; ++e) {
          float x = z[j + e];
          asm volatile("" : "+v"(x));
          f(j + e, x);
        }
      }
    }
  };
  unsigned khi = sample_wave_max(sample_key(hi)), klo = sample_wave_max(~sample_key(lo));
  if (lane == 0) {
    range[0][w] = khi;
    range[1][w] = klo;
  }
#pragma unroll
  for (int j = 0; j < PB; ++j) {
    bin_mass[tid + j * NT] = 0;
    bin_count[tid + j * NT] = 0;
  }
  if (tid < 2) n_listed[tid] = 0;
  if (tid == 0) upper = 0;
  __syncthreads();
  khi = sample_wave_max(lane < NT / 64 ? range[0][lane] : 0u);
  klo = sample_wave_max(lane < NT / 64 ? range[1][lane] : 0u);
  const float zmax = sample_unkey(khi);
  if (zmax == -INFINITY || set.greedy) {
    unsigned first = 0;   // complement of the lowest index of the largest logit
#pragma unroll
    for (int j = R - 1; j >= 0; --j)
      if (z[j] == zmax) first = ~(unsigned)(i0 + j);
    first = sample_wave_max(first);
    __syncthreads();
    if (lane == 0) range[0][w] = first;
    __syncthreads();
    first = ~sample_wave_max(lane < NT / 64 ? range[0][lane] : 0u);
    if (tid == 0) {
      if (zmax == -INFINITY) sample_answer(a, row, -1, -INFINITY);
      else sample_answer(a, row, (long)first, 0.f);
    }
    return;
  }
  SampleMass mass(zmax, set.y, 0);
  unsigned long long q[R];
  unsigned floored = 0;   // bit j: cut by min-p
  // masses of the codes from `least` on, then down to what their sum leaves room for: it is below (the sum of their upper 17 bits + V) 2^47
  auto weigh = [&](float least) {
#pragma unroll
    for (int j = 0; j < R; ++j) q[j] = 0;
    unsigned sum = 0;
    each([&](int j, float x) {
      if (x >= least) {
        const SampleMass::Power e = mass.power(x);
        q[j] = mass.whole(e);
        floored |= (mass.value(e) >= set.m ? 0u : 1u) << j;
        sum += (unsigned)(q[j] >> 47);
      }
    });
    sum = sample_wave_sum(sum);
    if (lane == 0) atomicAdd(&upper, sum);
    __syncthreads();
    mass.scale(max(17 - __builtin_clz((unsigned)__builtin_amdgcn_readfirstlane((int)upper) + (unsigned)V), 0));
#pragma unroll
    for (int j = 0; j < R; j += PAIR)
      if (j < steps)
#pragma unroll
        for (int e = 0; e < PAIR; ++e) q[j + e] >>= mass.down;
  };
  float t = sample_massless(zmax, set.y);
  unsigned r = 0;
  const bool by_mass = set.p < 1.0;
  if (by_mass) weigh(t);
  if (set.k < V || by_mass) {
    const SampleBins bins = sample_bins(zmax, sample_unkey(~klo), set.y, kSampleBins);
    each([&](int j, float x) {
      if (x > t) {
        const int b = bins.of(x);
        atomicAdd(&bin_count[b], 1u);
        if (by_mass && q[j]) atomicAdd(&bin_mass[b], q[j]);
      }
    });
    __syncthreads();
    unsigned long long m = 0, m_before, total;
    unsigned c = 0, c_before, c_all;
#pragma unroll
    for (int j = 0; j < PB; ++j) {
      m += bin_mass[tid * PB + j];
      c += bin_count[tid * PB + j];
    }
    sample_block_scan<NT>(blk, m, c, m_before, c_before, total, c_all);
    // codes of bin b above t into m_z, m_mass; their number
    auto list = [&](int b, int which) {
      each([&](int j, float x) {
        if (x > t && bins.of(x) == b) {
          const int to = atomicAdd(&n_listed[which], 1);
          if (to < 64) {
            m_z[to] = x;
            m_mass[to] = by_mass ? q[j] : 0ull;
          }
        }
      });
      __syncthreads();
      return n_listed[which];
    };
    // the smallest and largest key of bin b above t
    auto keys_of = [&](int b, unsigned& first, unsigned& last) {
      if (tid == 0) {
        key_range[0] = ~0u;
        key_range[1] = 0;
      }
      __syncthreads();
      unsigned l = ~0u, h = 0;
      each([&](int j, float x) {
        if (x > t && bins.of(x) == b) {
          l = min(l, sample_key(x));
          h = max(h, sample_key(x));
        }
      });
      if (h) {
        atomicMin(&key_range[0], l);
        atomicMax(&key_range[1], h);
      }
      __syncthreads();
      first = key_range[0];
      last = key_range[1];
    };
    int kb = kSampleBins;                          // the bin that top-k cuts
    unsigned long long k_above = 0, k_in = 0;      // mass before that bin, and in it above t
    unsigned long long qt = 0;                     // mass of a code at t
    if ((unsigned)set.k < c_all) {
      if (c_before < (unsigned)set.k && (unsigned)set.k <= c_before + c) {
        unsigned cr = c_before;
        unsigned long long mr = m_before;
#pragma unroll
        for (int j = 0; j < PB; ++j) {
          const unsigned n = bin_count[tid * PB + j];
          if (cr < (unsigned)set.k && (unsigned)set.k <= cr + n) {
            found.bin = tid * PB + j;
            found.count = (unsigned)set.k - cr;
            found.mass = mr;
          }
          cr += n;
          mr += bin_mass[tid * PB + j];
        }
      }
      __syncthreads();
      kb = found.bin;
      const unsigned want = found.count;
      k_above = found.mass;
      const int n = list(kb, 0);
      if (n <= 64) {
        if (w == 0) {
          const float mz = lane < n ? m_z[lane] : -INFINITY;
          unsigned gt = 0, ge = 0;
          for (int i = 0; i < n; ++i) {
            const float o = __uint_as_float(sample_lane(__float_as_uint(mz), i));
            gt += o > mz;
            ge += o >= mz;
          }
          const int at = __builtin_ctzll(__ballot(lane < n && gt < want && want <= ge));
          const float z_at = __uint_as_float(sample_lane(__float_as_uint(mz), at));
          const unsigned long long in = by_mass ? sample_wave_sum(mz > z_at ? m_mass[lane] : 0ull) : 0ull;
          if (lane == 0) {
            cut.t = z_at;
            cut.r = want - sample_lane(gt, at);
            cut.in = in;
          }
        }
        __syncthreads();
        t = cut.t;
        r = cut.r;
        k_in = cut.in;
      } else {
        unsigned first, last;
        keys_of(kb, first, last);
        unsigned long long before;
        const unsigned key = sample_search<NT>(blk, found, part, first, last, want, before, [&](auto f) {
          each([&](int j, float x) {
            if (x > t && bins.of(x) == kb) f(sample_key(x), [] { return 1ull; });
          });
        });
        t = sample_unkey(key);
        r = want - (unsigned)before;
        if (by_mass) {
          unsigned long long in = 0, none;
          unsigned none_c, none_all;
          each([&](int j, float x) {
            if (x > t && bins.of(x) == kb) in += q[j];
          });
          sample_block_scan<NT>(blk, in, 0u, none, none_c, k_in, none_all);
        }
      }
      if (by_mass) {
        qt = mass.q(t);
        total = k_above + k_in + r * qt;
      }
    }
    if (by_mass) {
      const unsigned long long bound = sample_bound(set.p, total);
      if (kb < kSampleBins && bound > k_above + k_in) {   // on the ties that top-k kept
        r = min(r, sample_ceil_div(bound - k_above - k_in, qt));
      } else {
        if (m_before < bound && bound <= m_before + m) {
#pragma unroll
          for (int j = 0; j < PB; ++j) {
            const unsigned long long n = bin_mass[tid * PB + j];
            if (m_before < bound && bound <= m_before + n) {
              found.bin = tid * PB + j;
              found.mass = m_before;
            }
            m_before += n;
          }
        }
        __syncthreads();
        const int pb = found.bin;
        const unsigned long long need = bound - found.mass;
        const int n = list(pb, 1);
        if (n <= 64) {
          if (w == 0) {
            const float mz = lane < n ? m_z[lane] : -INFINITY;
            const unsigned long long mq = lane < n ? m_mass[lane] : 0ull;
            unsigned long long gt = 0, ge = 0;
            for (int i = 0; i < n; ++i) {
              const float o = __uint_as_float(sample_lane(__float_as_uint(mz), i));
              const unsigned long long v = sample_lane(mq, i);
              gt += o > mz ? v : 0ull;
              ge += o >= mz ? v : 0ull;
            }
            const int at = __builtin_ctzll(__ballot(lane < n && gt < need && need <= ge));
            if (lane == at) {
              cut.t = mz;
              cut.r = sample_ceil_div(need - gt, mq);
            }
          }
          __syncthreads();
          t = cut.t;
          r = cut.r;
        } else {
          unsigned first, last;
          keys_of(pb, first, last);
          unsigned long long before;
          const unsigned key = sample_search<NT>(blk, found, part, first, last, need, before, [&](auto f) {
            each([&](int j, float x) {
              if (x > t && bins.of(x) == pb) f(sample_key(x), [&] { return q[j]; });
            });
          });
          t = sample_unkey(key);
          r = sample_ceil_div(need - before, mass.q(t));
        }
      }
    }
  }
  if (!by_mass) weigh(t);   // (of what top-k kept alone)
  unsigned at_t = 0;
  unsigned long long sum = 0;
  const unsigned long long qt = r ? mass.q(t, set.m) : 0ull;
  each([&](int j, float x) {
    at_t += x == t && r > 0;
    sum += x > t && !(floored >> j & 1) ? q[j] : 0ull;
  });
  unsigned long long run, above;
  unsigned seen, all_t;
  sample_block_scan<NT>(blk, sum, at_t, run, seen, above, all_t);
  const unsigned long long total = above + min(all_t, r) * qt, target = sample_target(set.u, total);
  run += min(seen, r) * qt;
  const unsigned long long here = sum + (min(seen + at_t, r) - min(seen, r)) * qt;
  if (run <= target && target < run + here) {
    int at = 0;
    float z_at = 0.f;
    bool drawn = false;
    each([&](int j, float x) {
      const bool tie = x == t && r > 0;
      if (x > t && !(floored >> j & 1)) run += q[j];
      if (tie && seen < r) run += qt;
      seen += tie;
      if (!drawn && run > target) {
        drawn = true;
        at = j;
        z_at = x;
      }
    });
    sample_answer(a, row, i0 + at, mass.logp(z_at, total));
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The longest rows, a workgroup per chunk of 16384 codes: (1) largest and smallest logit of every chunk, (2) its bins, (3) the bins summed
// over the chunks, (4) the cuts' bins found, (5) the codes of those bins ("members") listed, equal ones of a chunk as one where they are
// many, and the mass of what every chunk keeps whole, (6) one workgroup per row: the cuts among the members, the chunk that the draw falls
// into, and the code in it.  Three passes over the logits, of which the cache serves the later two; nobody waits for another workgroup
// inside a kernel.
//
// Where both cuts are on, what top-k keeps of its bin is not known before its members are looked at; the mass that top-p cuts at is then
// known only to within that bin's mass, and the members of all bins it can fall into are taken.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSampleChunkThreads = 1024, kSampleChunkIpt = 16, kSampleChunk = kSampleChunkThreads * kSampleChunkIpt;
constexpr int kSampleMaxChunks = 1024;          // V <= 2^24
constexpr int kSampleFewChunks = 4;             // up to which the bins are summed where the cuts are found (500 rows of 50000, all cuts: 150
                                                // us, 164 with a launch of its own; one row of 130000, eight chunks, 46 and 45)
constexpr int kSampleHere = 2048;               // members of a chunk listed one by one; with more, equal ones as one
constexpr int kSampleMembers = 4096;            // members of a row that the last kernel holds in LDS

// Bins of such a row: 128 to a power of two of 1 + s (max z - z), eight powers down to where nothing has mass (62 / y) or the smallest
// logit.  Next to the largest logit they are 30 times as fine as linear ones (logits that hardly differ, beside masks of the type's lowest
// value, would all lie in one of those), where a cut of ordinary logits falls twice as coarse.  Sum, product and the bits of a positive fp32 are monotone; a NaN goes to the last bin.
struct SampleLogBins {
  float zmax, s;
  __device__ __forceinline__ int of(float z) const {
    const unsigned bits = __float_as_uint(fmaf(zmax - z, s, 1.f)) - 0x3F800000u;
    return (int)min(bits >> 16, (unsigned)kSampleBins - 1);
  }
};
__device__ __forceinline__ SampleLogBins sample_log_bins(float zmax, float zmin, double y) {
  const float d = fminf(zmax - zmin, (float)fmin(fmax(62.0 / y, 1e-36), 3e38));
  return SampleLogBins{zmax, d > 0.f && zmax < INFINITY ? fminf(255.f / d, 3e38f) : 0.f};
}

struct SampleState {                   // of a row
  float zmax, zmin;
  unsigned first;                      // lowest index of the largest logit
  int down;                            // of its masses
  int kb;                              // the bin that top-k cuts; kSampleBins: none
  unsigned want;                       // codes kept of it
  int b0, b1;                          // bins that the last cut falls into; kSampleBins: no cut
  int fb;                              // the first bin with codes that min-p cuts; bins before min(b0, fb) are kept whole
  int n_members;
  unsigned long long above, base;      // mass before kb, and before b0
  unsigned long long bound;            // the mass that top-p cuts at, where top-k cuts nothing
  float lo[3], hi[3];                  // logits of bins b0 .. b1, of kb, and of fb if it is before b0 (lo > hi: none)
};

struct SampleLong {
  long row0;                           // first row of the batch
  int chunks;
  int uncut;                           // no row has a cut: state is not there
  int most;                            // members that a row's list holds (with more the last kernel searches the row itself)
  unsigned long long* best;            // [row][chunk] key of the largest logit << 32 | ~lowest index that holds it
  unsigned* least;                     // [row][chunk] ~key of the smallest logit that is not -inf
  float* sum;                          // [row][chunk] sum of 2^(log2 e - the chunk's largest), roughly
  int* floor;                          // [row][chunk] first bin with a code that min-p cuts
  unsigned long long* mass;            // [row][chunk][bin]
  unsigned* count;
  unsigned long long* row_mass;        // [row][bin]
  unsigned* row_count;
  SampleState* state;                  // [row]
  unsigned long long* chunk_mass;      // [row][chunk] of codes kept whole
  float* m_z;                          // [row][most] logit
  unsigned* m_where;                   // its chunk << 15 | how many (1 .. 16384)
};

template <typename T>
__device__ __forceinline__ void sample_load_chunk(const SampleArgs& a, const T* logits, int i0, float (&z)[kSampleChunkIpt]) {
  if (i0 + kSampleChunk <= a.V) {
    const T* p = logits + i0 + threadIdx.x;
#pragma unroll
    for (int j = 0; j < kSampleChunkIpt; ++j) {
      const float x = GroupNum<T>::get(p[j * kSampleChunkThreads]);
      z[j] = x == x ? x : -INFINITY;
    }
  } else {
#pragma unroll
    for (int j = 0; j < kSampleChunkIpt; ++j) z[j] = sample_logit(logits, i0 + j * kSampleChunkThreads + (int)threadIdx.x, a.V);
  }
}

// 2^((z - top) log2(e) / T) in 32 bits, never below what it stands for by more than 2^-14 of itself: the difference in halves (that of two fp32
// may be infinite), y2 = twice the factor (a tiny one may be 0, a huge one is cut off), and 1 where that is no number (0 inf, inf - inf)
__device__ __forceinline__ float sample_rough(float z, float top, float y2) {
  return __builtin_amdgcn_exp2f(fminf(fmaf(z, 0.5f, -0.5f * top) * y2, 0.f));
}
__device__ __forceinline__ float sample_rough_factor(double y) { return 2.f * (float)fmin(y, 1.5e38); }

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_range_kernel(SampleArgs a, SampleLong l) {
  __shared__ unsigned sh[3][kSampleChunkThreads / 64];
  __shared__ float sh_sum[kSampleChunkThreads / 64];
  const long r = blockIdx.x / l.chunks;
  const SampleRow set = sample_row(a, l.row0 + r);
  const int c = blockIdx.x - (int)(r * l.chunks), i0 = c * kSampleChunk, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  float z[kSampleChunkIpt], hi = -INFINITY, lo = INFINITY;
  sample_load_chunk(a, reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride, i0, z);
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    hi = fmaxf(hi, z[j]);
    lo = fminf(lo, z[j] > -INFINITY ? z[j] : INFINITY);
  }
  unsigned at = 0;
#pragma unroll
  for (int j = kSampleChunkIpt - 1; j >= 0; --j)
    if (z[j] == hi) at = ~(unsigned)(i0 + j * kSampleChunkThreads + (int)threadIdx.x);
  const unsigned top = sample_wave_max(sample_key(hi));
  at = sample_wave_max(sample_key(hi) == top ? at : 0u);
  const unsigned least = sample_wave_max(~sample_key(lo));
  if (lane == 0) {
    sh[0][w] = top;
    sh[1][w] = at;
    sh[2][w] = least;
  }
  __syncthreads();
  const bool in = lane < kSampleChunkThreads / 64;
  const unsigned t = in ? sh[0][lane] : 0u, all = sample_wave_max(t);
  // the chunk's sum next to its largest logit: every row's masses are scaled by its own
  float sum = 0.f;
  if (!set.greedy) {
    const float best = sample_unkey(all), y2 = sample_rough_factor(set.y);
#pragma unroll
    for (int j = 0; j < kSampleChunkIpt; ++j) sum += sample_rough(z[j], best, y2);
    sum = sample_wave_sum(sum);
    if (lane == 0) sh_sum[w] = sum;
    __syncthreads();
  }
  if (w == 0) {
    sum = sample_wave_sum(in && !set.greedy ? sh_sum[lane] : 0.f);
    const unsigned i = sample_wave_max(in && t == all ? sh[1][lane] : 0u), s = sample_wave_max(in ? sh[2][lane] : 0u);
    if (lane == 0) {
      l.best[r * l.chunks + c] = (unsigned long long)all << 32 | i;
      l.least[r * l.chunks + c] = s;
      l.sum[r * l.chunks + c] = sum;
    }
  }
}

struct SampleRange {
  float zmax, zmin;
  unsigned first;
  int down;
};
// the row's range from its chunks', and how far its masses go down: the row's sum is below 2^(down + 1) times the largest, so that of the masses
// below 2^62.  y: log2(e) / T.  Every thread.  Ends with a barrier.  (In the same order in every kernel: the same number.)
__device__ __forceinline__ SampleRange sample_range(const SampleLong& l, long r, double y, unsigned* sh) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const float y2 = sample_rough_factor(y);
    unsigned top = kSampleKeyMasked, at = 0, least = 0;
    float sum = 0.f;   // next to `top`
    for (int c = lane; c < l.chunks; c += 64) {
      const unsigned long long b = l.best[r * l.chunks + c];
      const unsigned t = (unsigned)(b >> 32);
      const float was = sample_unkey(top), z = sample_unkey(t), best = fmaxf(was, z);
      at = t > top ? (unsigned)b : (t == top ? max(at, (unsigned)b) : at);
      top = max(top, t);
      least = max(least, l.least[r * l.chunks + c]);
      sum = sum * sample_rough(was, best, y2) + l.sum[r * l.chunks + c] * sample_rough(z, best, y2);
    }
    const unsigned all = sample_wave_max(top);
    at = sample_wave_max(top == all ? at : 0u);
    least = sample_wave_max(least);
    sum = sample_wave_sum(sum * sample_rough(sample_unkey(top), sample_unkey(all), y2));
    if (lane == 0) {
      sh[0] = all;
      sh[1] = ~least;
      sh[2] = ~at;
      sh[3] = (unsigned)max((int)(__float_as_uint(sum * 1.01f) >> 23) - 127, 0);
    }
  }
  __syncthreads();
  return SampleRange{sample_unkey(sh[0]), sample_unkey(sh[1]), sh[2], (int)sh[3]};
}

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_bins_kernel(SampleArgs a, SampleLong l) {
  __shared__ unsigned long long bin_mass[kSampleBins];
  __shared__ unsigned bin_count[kSampleBins];
  __shared__ unsigned sh[4];
  __shared__ int floor;
  static_assert(kSampleBins == kSampleChunkThreads, "a thread owns a bin");
  const long r = blockIdx.x / l.chunks;
  const int c = blockIdx.x - (int)(r * l.chunks), tid = threadIdx.x;
  const SampleRow set = sample_row(a, l.row0 + r);
  float z[kSampleChunkIpt];
  sample_load_chunk(a, reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride, c * kSampleChunk, z);
  bin_mass[tid] = 0;
  bin_count[tid] = 0;
  if (tid == 0) floor = kSampleBins;
  const SampleRange g = sample_range(l, r, set.y, sh);   // (its barrier: the bins are cleared)
  if (g.zmax == -INFINITY || set.greedy) return;
  const SampleMass mass(g.zmax, set.y, g.down);
  const SampleLogBins bins = sample_log_bins(g.zmax, g.zmin, set.y);
  const bool by_count = set.k < a.V, by_floor = set.m > 0.0;
  int first = kSampleBins;
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    const int b = bins.of(z[j]);
    const SampleMass::Power e = mass.power(z[j]);
    const unsigned long long q = mass.whole(e);
    if (q) {
      if (by_count) atomicAdd(&bin_count[b], 1u);
      atomicAdd(&bin_mass[b], q);
    }
    if (by_floor) first = min(first, mass.value(e) >= set.m || z[j] == -INFINITY ? kSampleBins : b);
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
  }
  if (first < kSampleBins) atomicMin(&floor, first);
  __syncthreads();
  const size_t o = ((size_t)r * l.chunks + c) * kSampleBins + tid;
  l.mass[o] = bin_mass[tid];
  l.count[o] = bin_count[tid];
  if (tid == 0) l.floor[r * l.chunks + c] = floor;
}

// Where no row has a cut the mass of every chunk is all that the last kernel needs: three launches (one row of 50000 fp32 22 us, 16 of 2^20
// 50; with bins, cuts and members all the same 33 and 73).
template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_mass_kernel(SampleArgs a, SampleLong l) {
  __shared__ unsigned sh[4];
  __shared__ unsigned long long part[kSampleChunkThreads / 64];
  const long r = blockIdx.x / l.chunks;
  const int c = blockIdx.x - (int)(r * l.chunks), lane = threadIdx.x & 63;
  const SampleRow set = sample_row(a, l.row0 + r);
  float z[kSampleChunkIpt];
  sample_load_chunk(a, reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride, c * kSampleChunk, z);
  const SampleRange g = sample_range(l, r, set.y, sh);
  if (g.zmax == -INFINITY || set.greedy) return;
  const SampleMass mass(g.zmax, set.y, g.down);
  unsigned long long sum = 0;
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    sum += mass.q(z[j]);
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
  }
  sum = sample_wave_sum(sum);
  if (lane == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x < 64) {
    sum = sample_wave_sum(lane < kSampleChunkThreads / 64 ? part[lane] : 0ull);
    if (lane == 0) l.chunk_mass[r * l.chunks + c] = sum;
  }
}

// bins summed over the chunks: a workgroup owns 64 bins of a row, its 16 waves every 16th chunk
__global__ void __launch_bounds__(1024) sample_sum_bins_kernel(SampleLong l) {
  __shared__ unsigned long long mass[16][64];
  __shared__ unsigned count[16][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const long r = blockIdx.x / (kSampleBins / 64);
  const int b = (int)(blockIdx.x % (kSampleBins / 64)) * 64 + lane;
  unsigned long long m = 0;
  unsigned n = 0;
  for (int c = w; c < l.chunks; c += 16) {
    const size_t o = ((size_t)r * l.chunks + c) * kSampleBins + b;
    m += l.mass[o];
    n += l.count[o];
  }
  mass[w][lane] = m;
  count[w][lane] = n;
  __syncthreads();
  if (w == 0) {
    for (int v = 1; v < 16; ++v) {
      m += mass[v][lane];
      n += count[v][lane];
    }
    l.row_mass[r * kSampleBins + b] = m;
    l.row_count[r * kSampleBins + b] = n;
  }
}

// the cuts' bins of a row, a thread per bin (a kernel of its own: finding them by the last workgroup of the one above needs a fence that
// empties the L2, measured 30 us against 5 + 5)
__global__ void __launch_bounds__(1024) sample_cuts_kernel(SampleArgs a, SampleLong l) {
  constexpr int NT = 1024;
  __shared__ SampleBlock<NT> blk;
  __shared__ SampleState st;
  __shared__ unsigned sh[4];
  const int tid = threadIdx.x;
  const long r = blockIdx.x;
  const SampleRow set = sample_row(a, l.row0 + r);
  const SampleRange g = sample_range(l, r, set.y, sh);
  if (tid == 0) {
    st.zmax = g.zmax;
    st.zmin = g.zmin;
    st.first = g.first;
    st.down = g.down;
    st.kb = st.b0 = st.b1 = st.fb = kSampleBins;
    st.want = 0;
    st.n_members = 0;
    st.above = st.base = st.bound = 0;
  }
  __syncthreads();
  if (g.zmax > -INFINITY && !set.greedy) {
    unsigned long long m = 0;
    unsigned n = 0;
    if (l.chunks <= kSampleFewChunks) {
#pragma unroll
      for (int c = 0; c < kSampleFewChunks; ++c) {
        if (c < l.chunks) {
          const size_t o = ((size_t)r * l.chunks + c) * kSampleBins + tid;
          m += l.mass[o];
          n += l.count[o];
        }
      }
    } else {
      m = l.row_mass[r * kSampleBins + tid];
      n = l.row_count[r * kSampleBins + tid];
    }
    int f = kSampleBins;
    for (int c = tid; c < l.chunks; c += NT) f = min(f, l.floor[r * l.chunks + c]);
    if (f < kSampleBins) atomicMin(&st.fb, f);
    unsigned long long m_before, m_all;
    unsigned c_before, c_all;
    sample_block_scan<NT>(blk, m, n, m_before, c_before, m_all, c_all);
    if (set.k < a.V && c_before < (unsigned)set.k && (unsigned)set.k <= c_before + n && (unsigned)set.k < c_all) {
      st.kb = st.b0 = st.b1 = tid;
      st.want = (unsigned)set.k - c_before;
      st.above = st.base = m_before;
      st.bound = m;                    // (of kb, until the lines below have read it)
    }
    __syncthreads();
    if (set.p < 1.0) {
      const bool cut = st.kb < kSampleBins;
      const unsigned long long lo = sample_bound(set.p, cut ? st.above : m_all), hi = sample_bound(set.p, cut ? st.above + st.bound : m_all);
      __syncthreads();
      if (m_before < lo && lo <= m_before + m) {
        st.b0 = tid;
        st.base = m_before;
      }
      if (m_before < hi && hi <= m_before + m) st.b1 = tid;
      if (tid == 0) st.bound = lo;
    }
  }
  __syncthreads();
  if (tid < 6) {   // the ends of the members' logits: the bins are monotone, so each is found bit by bit over the keys
    const SampleLogBins bins = sample_log_bins(g.zmax, g.zmin, set.y);
    const unsigned massless = sample_key(sample_massless(g.zmax, set.y));
    const int which = tid >> 1;
    const int x = which == 0 ? st.b0 : which == 1 ? st.kb : st.fb, y = which == 0 ? st.b1 : x;
    unsigned key = 0;   // tid even: the largest key whose bin is behind y (lo is the one above it); odd: the largest whose bin is x or behind it
    for (int b = 31; b >= 0; --b) {
      const unsigned c = key | 1u << b;
      const float z = sample_unkey(c);
      const bool behind = c <= kSampleKeyMasked || (z <= g.zmax && bins.of(z) >= (tid & 1 ? x : y + 1));
      if (behind) key = c;
    }
    const bool none = x >= kSampleBins || (which == 2 && st.fb >= st.b0);
    if (tid & 1) st.hi[which] = none ? -INFINITY : sample_unkey(key);
    else st.lo[which] = none ? INFINITY : sample_unkey(max(key, massless) + 1);
  }
  __syncthreads();
  if (tid == 0) l.state[r] = st;
}

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_members_kernel(SampleArgs a, SampleLong l) {
  constexpr int NT = kSampleChunkThreads, LOOKS = 16;
  constexpr unsigned EMPTY = kSampleKeyMasked;                // (-inf is no member)
  __shared__ SampleBlock<NT> blk;
  __shared__ unsigned m_key[kSampleHere], m_count[kSampleHere];
  __shared__ int n_here, first_here;
  const long r = blockIdx.x / l.chunks;
  const int c = blockIdx.x - (int)(r * l.chunks), i0 = c * kSampleChunk, tid = threadIdx.x, lane = tid & 63;
  const SampleRow set = sample_row(a, l.row0 + r);
  const SampleState st = l.state[r];
  if (st.zmax == -INFINITY || set.greedy) return;
  const bool any = st.b0 < kSampleBins || st.fb < kSampleBins;
  float z[kSampleChunkIpt];
  unsigned is = 0;   // bit j: z[j] is a member
  if (any) {
    sample_load_chunk(a, reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride, i0, z);
#pragma unroll
    for (int j = 0; j < kSampleChunkIpt; ++j) is |= (unsigned)(z[j] >= st.lo[0] && z[j] <= st.hi[0]) << j;
    if ((st.kb < st.b0 || st.kb > st.b1) && st.kb < kSampleBins) {
#pragma unroll
      for (int j = 0; j < kSampleChunkIpt; ++j) is |= (unsigned)(z[j] >= st.lo[1] && z[j] <= st.hi[1]) << j;
    }
    if (st.fb < st.b0) {
#pragma unroll
      for (int j = 0; j < kSampleChunkIpt; ++j) is |= (unsigned)(z[j] >= st.lo[2] && z[j] <= st.hi[2]) << j;
    }
  }
  // what the chunk keeps whole: its bins before the cuts
  const unsigned long long m = tid < min(st.b0, st.fb) ? l.mass[((size_t)r * l.chunks + c) * kSampleBins + tid] : 0ull;
  unsigned long long before, all;
  unsigned c_before, n;
  sample_block_scan<NT>(blk, m, (unsigned)__builtin_popcount(is), before, c_before, all, n);
  if (tid == 0) {
    l.chunk_mass[r * l.chunks + c] = all;
    if (n > 0 && n <= kSampleHere) first_here = atomicAdd(&l.state[r].n_members, (int)n);
    n_here = 0;
  }
  if (n == 0) return;
  float* const out_z = l.m_z + r * l.most;
  unsigned* const out_where = l.m_where + r * l.most;
  const unsigned chunk = (unsigned)c << 15;
  auto put = [&](int to, float x, unsigned count) {
    if (to < l.most) {
      out_z[to] = x;
      out_where[to] = chunk | count;
    }
  };
  __syncthreads();
  if (n <= kSampleHere) {
    if (is) {
      int to = first_here + (int)c_before;
#pragma unroll
      for (int j = 0; j < kSampleChunkIpt; ++j)
        if (is >> j & 1) put(to++, z[j], 1);
    }
    return;
  }
  // many: counted by key in a table of the workgroup; what finds no room there goes into the list as it is
  for (int i = tid; i < kSampleHere; i += NT) {
    m_key[i] = EMPTY;
    m_count[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    unsigned long long todo = __ballot(is >> j & 1);
    const unsigned key = sample_key(z[j]);
    for (int look = 0; todo && look < 2; ++look) {   // (keys that several lanes hold go in as one)
      const int lead = __builtin_ctzll(todo);
      const unsigned long long same = todo & __ballot((is >> j & 1) && key == sample_lane(key, lead));
      if (__builtin_popcountll(same) == 1 && look) break;
      bool in = false;
      if (lane == lead) {
        const unsigned h = (key * 2654435761u) >> 21;
        for (int i = 0; i < LOOKS && !in; ++i) {
          const unsigned at = (h + i) & (kSampleHere - 1), old = atomicCAS(&m_key[at], EMPTY, key);
          if (old == EMPTY || old == key) {
            atomicAdd(&m_count[at], (unsigned)__builtin_popcountll(same));
            in = true;
          }
        }
        if (!in) put(atomicAdd(&l.state[r].n_members, 1), z[j], (unsigned)__builtin_popcountll(same));
      }
      todo &= ~same;
    }
    if (todo >> lane & 1) {
      bool in = false;
      const unsigned h = (key * 2654435761u) >> 21;
      for (int i = 0; i < LOOKS && !in; ++i) {
        const unsigned at = (h + i) & (kSampleHere - 1), old = atomicCAS(&m_key[at], EMPTY, key);
        if (old == EMPTY || old == key) {
          atomicAdd(&m_count[at], 1u);
          in = true;
        }
      }
      if (!in) put(atomicAdd(&l.state[r].n_members, 1), z[j], 1);
    }
  }
  __syncthreads();
  int mine = 0;
  for (int i = tid; i < kSampleHere; i += NT) mine += m_count[i] > 0;
  int to = mine ? atomicAdd(&n_here, mine) : 0;
  __syncthreads();
  if (tid == 0 && n_here) first_here = atomicAdd(&l.state[r].n_members, n_here);
  __syncthreads();
  to += first_here;
  for (int i = tid; i < kSampleHere; i += NT)
    if (m_count[i] > 0) put(to++, sample_unkey(m_key[i]), m_count[i]);
}

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_finish_kernel(SampleArgs a, SampleLong l) {
  constexpr int NT = kSampleChunkThreads;
  __shared__ SampleBlock<NT> blk;
  __shared__ SampleFound found;
  __shared__ unsigned long long part[kSampleBins];
  __shared__ float m_z[kSampleMembers];
  __shared__ unsigned m_where[kSampleMembers];
  __shared__ unsigned long long chunk[kSampleMaxChunks];
  __shared__ unsigned chunk_ties[kSampleMaxChunks];
  __shared__ unsigned key_range[2], sh_range[4];
  __shared__ int sh_chunk;
  __shared__ unsigned sh_tied;
  __shared__ unsigned long long sh_before;
  const long r = blockIdx.x, row = l.row0 + r;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const SampleRow set = sample_row(a, row);
  SampleState st{};
  if (l.uncut) {
    const SampleRange g = sample_range(l, r, set.y, sh_range);
    st.zmax = g.zmax;
    st.zmin = g.zmin;
    st.first = g.first;
    st.down = g.down;
    st.kb = st.b0 = st.b1 = st.fb = kSampleBins;
  } else {
    st = l.state[r];
  }
  if (st.zmax == -INFINITY || set.greedy) {
    if (tid == 0) {
      if (st.zmax == -INFINITY) sample_answer(a, row, -1, -INFINITY);
      else sample_answer(a, row, (long)st.first, 0.f);
    }
    return;
  }
  const SampleMass mass(st.zmax, set.y, st.down);
  const SampleLogBins bins = sample_log_bins(st.zmax, st.zmin, set.y);
  const T* logits = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const bool listed = st.n_members <= l.most, held = st.n_members <= kSampleMembers;   // (else the row itself is the list)
  const int n = listed ? st.n_members : a.V;
  const float massless = sample_massless(st.zmax, set.y);
  chunk[tid] = listed && tid < l.chunks ? l.chunk_mass[r * l.chunks + tid] : 0ull;
  chunk_ties[tid] = 0;
  if (tid == 0) {
    key_range[0] = ~0u;
    key_range[1] = 0;
    sh_chunk = 0;   // (logits that change during the call: some chunk of the row all the same)
    sh_before = 0;
    sh_tied = 0;
  }
  __syncthreads();
  // f(logit, how many, chunk) for every member
  auto each = [&](auto f) {
    if (held) {
      for (int i = tid; i < n; i += NT) f(m_z[i], m_where[i] & 0x7FFFu, m_where[i] >> 15);
    } else {
#pragma unroll 1
      for (int i = tid; i < n; i += NT) {
        const float z = listed ? l.m_z[r * l.most + i] : sample_logit(logits, i, a.V);
        const unsigned at = listed ? l.m_where[r * l.most + i] : (unsigned)(i / kSampleChunk) << 15 | 1u;
        if (z > massless) f(z, at & 0x7FFFu, at >> 15);
      }
    }
  };
  // the members' keys: fewer bits to search
  unsigned lo = 0, hi = 0;   // lo: complemented
  if (held) {
    for (int i = tid; i < n; i += NT) {
      m_z[i] = l.m_z[r * l.most + i];
      m_where[i] = l.m_where[r * l.most + i];
    }
  }
  each([&](float z, unsigned, unsigned) {   // (a thread reads what it wrote)
    lo = max(lo, ~sample_key(z));
    hi = max(hi, sample_key(z));
  });
  lo = sample_wave_max(lo);
  hi = sample_wave_max(hi);
  if (lane == 0 && hi) {
    atomicMin(&key_range[0], ~lo);
    atomicMax(&key_range[1], hi);
  }
  __syncthreads();
  const unsigned kmin = key_range[0], kmax = key_range[1];
  float t = massless;
  unsigned ties = 0;   // codes kept of those at t
  unsigned long long qt = 0, before, all = 0;
  unsigned none, none_all;
  unsigned long long total = 0;
  if (st.kb < kSampleBins) {
    const unsigned key = sample_search<NT>(blk, found, part, kmin, kmax, st.want, before, [&](auto f) {
      each([&](float z, unsigned c, unsigned) {
        if (bins.of(z) == st.kb) f(sample_key(z), [&] { return (unsigned long long)c; });
      });
    });
    t = sample_unkey(key);
    ties = st.want - (unsigned)before;
    qt = mass.q(t);
    unsigned long long in = 0;
    each([&](float z, unsigned c, unsigned) {
      if (z > t && bins.of(z) == st.kb) in += c * mass.q(z);
    });
    sample_block_scan<NT>(blk, in, 0u, before, none, all, none_all);
    total = st.above + all + ties * qt;
  }
  if (set.p < 1.0) {
    const unsigned long long bound = st.kb < kSampleBins ? sample_bound(set.p, total) : st.bound;
    // (bins from b0 on; those behind b1, if any, are not reached)
    if (st.kb < kSampleBins && bound > st.above + all) {   // on the ties that top-k kept
      ties = min(ties, sample_ceil_div(bound - st.above - all, qt));
    } else {
      const unsigned key = sample_search<NT>(blk, found, part, kmin, kmax, bound - st.base, before, [&](auto f) {
        each([&](float z, unsigned c, unsigned) {
          if (z > t && bins.of(z) >= st.b0) f(sample_key(z), [&] { return c * mass.q(z); });
        });
      });
      t = sample_unkey(key);
      ties = sample_ceil_div(bound - st.base - before, mass.q(t));
    }
  }
  qt = ties ? mass.q(t, set.m) : 0ull;
  // kept members into their chunks, and the ties at t
  each([&](float z, unsigned c, unsigned at) {
    if (z > t) {
      const unsigned long long q = mass.q(z, set.m);
      if (q) atomicAdd(&chunk[at], c * q);
    }
    if (z == t && ties) atomicAdd(&chunk_ties[at], c);
  });
  __syncthreads();
  unsigned tied, tied_all;
  const unsigned at_chunk = chunk_ties[tid];
  sample_block_scan<NT>(blk, 0ull, at_chunk, before, tied, all, tied_all);
  const unsigned long long mine = chunk[tid] + min(at_chunk, ties > tied ? ties - tied : 0u) * qt;
  sample_block_scan<NT>(blk, mine, 0u, before, none, total, none_all);
  const unsigned long long target = sample_target(set.u, total);
  if (before <= target && target < before + mine) {
    sh_chunk = tid;
    sh_before = before;
    sh_tied = tied;
  }
  __syncthreads();
  // ... and in that chunk, 16 neighbouring codes per thread.  Where few of them are kept these are listed first, in their order (the members
  // are done with), and shared out anew: an exponential for every step in which one of a wave's 64 codes is kept would take longer
  const int i0 = sh_chunk * kSampleChunk, mine0 = tid * kSampleChunkIpt;
  float z[kSampleChunkIpt];
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; j += 4) {
    const int i = i0 + mine0 + j;
    if (i + 4 <= a.V) {
      GroupUnit<T, 4> u;
      u.load(logits + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float x = GroupNum<T>::get(u.v[e]);
        z[j + e] = x == x ? x : -INFINITY;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) z[j + e] = sample_logit(logits, i + e, a.V);
    }
  }
  unsigned is = 0;
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) is |= (unsigned)(z[j] > t || (z[j] == t && ties > 0)) << j;
  unsigned first, kept;
  sample_block_scan<NT>(blk, 0ull, (unsigned)__builtin_popcount(is), before, first, all, kept);
  if (kept <= kSampleMembers) {
#pragma unroll
    for (int j = 0; j < kSampleChunkIpt; ++j) {
      if (is >> j & 1) {
        m_z[first] = z[j];
        m_where[first++] = (unsigned)(mine0 + j);
      }
    }
    __syncthreads();
    constexpr int N = kSampleMembers / NT;
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = tid * N + j < (int)kept ? m_z[tid * N + j] : -INFINITY;
    sample_draw<NT>(a, row, x, [&](int j) { return i0 + (int)m_where[tid * N + j]; }, mass, set.m, t, ties, qt, blk, sh_before, sh_tied, target, total);
  } else {
    sample_draw<NT>(a, row, z, [&](int j) { return i0 + mine0 + j; }, mass, set.m, t, ties, qt, blk, sh_before, sh_tied, target, total);
  }
}

}  // namespace qinco
