// Sampling codes from logits: temperature, top-k, top-p and min-p, one given random number per row.
//
// MATHEMATICS.  Order the row's codes by (logit descending, index ascending); e_i = exp((z_i - max z) / T).  All three cuts keep a
// prefix of that order (top-k: its first k; top-p: every code with less than p of the kept mass before it; min-p: e_i >= min_p), so the
// kept set is {z > t} and the first r codes, by index, of those with z == t.  t and r are found by a radix selection over the logit's
// bits, by counts for top-k and by mass for top-p; nothing is sorted.  The code is the lowest kept index at which the running kept mass
// passes u times its total.
//
// NUMBERS.  A random number next to a border between two codes must fall on the side that exact arithmetic gives it, whatever order
// the sums are taken in: e is computed in 64 bits and held as a whole number of 2^-F, F = min(51, 62 - log2 V), and all sums are of
// whole numbers (atomics in any order give the same bits).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "group_kernel.hpp"   // GroupNum: conversions of the row types

namespace qinco {

constexpr unsigned kSampleKeyMasked = 0x007FFFFFu;   // sample_key(-inf): neither it nor NaN is ever drawn

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
  int F;
};

// fp32 -> unsigned, order-preserving; -0 counts as +0, NaN as -inf
__device__ __forceinline__ unsigned sample_key(float x) {
  if (x != x) return kSampleKeyMasked;
  const unsigned b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float sample_unkey(unsigned k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu)); }

// the row's settings, with every switched-off cut in the form that keeps everything
struct SampleRow {
  double invT, p, m, u;
  int k;
  bool greedy;
};

__device__ __forceinline__ SampleRow sample_row(const SampleArgs& a, long r) {
  SampleRow s;
  const double T = a.T_rows ? (double)a.T_rows[r] : a.T;
  s.greedy = !(T > 0.0);
  s.invT = s.greedy ? 0.0 : 1.0 / T;
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

// (z - max z) / T of a key; at or below the cut that rounds to a mass of zero
__device__ __forceinline__ double sample_arg(unsigned key, unsigned max_key, double zmax, double invT) {
  if (key == max_key) return 0.0;
  return fmax(((double)sample_unkey(key) - zmax) * invT, -100.0);
}
// e = exp(x) as a whole number of 2^-F (scale = 2^F <= 2^51: the sum with 2^52 rounds it to one, ties to even)
__device__ __forceinline__ unsigned long long sample_whole(double e, double scale) {
  return (unsigned long long)__double_as_longlong(fma(e, scale, 0x1p52)) & ((1ull << 52) - 1);
}
// exp(x) for -100 <= x <= 0: x = k ln 2 + r with |r| <= ln 2 / 2, the series of exp(r) to the 12th power (what is left out is below
// r^13 / 13! = 2e-16), times 2^k.  No range checks: sample_arg() keeps x inside.
__device__ __forceinline__ double sample_exp(double x) {
  const double k = rint(x * 1.4426950408889634074);
  double r = fma(k, -0x1.62e42fefa39efp-1, x);   // ln 2 in two parts
  r = fma(k, -0x1.abc9e3b39803fp-56, r);
  double e = 1.0 / 479001600.0;
  e = fma(e, r, 1.0 / 39916800.0);
  e = fma(e, r, 1.0 / 3628800.0);
  e = fma(e, r, 1.0 / 362880.0);
  e = fma(e, r, 1.0 / 40320.0);
  e = fma(e, r, 1.0 / 5040.0);
  e = fma(e, r, 1.0 / 720.0);
  e = fma(e, r, 1.0 / 120.0);
  e = fma(e, r, 1.0 / 24.0);
  e = fma(e, r, 1.0 / 6.0);
  e = fma(e, r, 0.5);
  e = fma(e, r, 1.0);
  e = fma(e, r, 1.0);
  return ldexp(e, (int)k);
}
// ... zero for what min-p cuts
__device__ __forceinline__ unsigned long long sample_mass(double x, double scale, double m) {
  const double e = sample_exp(x);
  return e >= m ? sample_whole(e, scale) : 0ull;
}

// smallest whole number that is at least p * total: "mass before < p * total" is "mass before < this"
__device__ __forceinline__ unsigned long long sample_bound(double p, unsigned long long total) {
  const double b = ceil(p * (double)total);
  const unsigned long long v = (unsigned long long)b;
  return v < 1 ? 1 : (v > total ? total : v);
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

// smallest r with r q >= rem (q >= 1, r < 2^25)
__device__ __forceinline__ unsigned sample_ceil_div(unsigned long long rem, unsigned long long q) {
  unsigned r = (unsigned)((double)rem / (double)q);
  while (r * q < rem) ++r;
  while (r && (r - 1) * q >= rem) --r;
  return r;
}

// Bins of the first look at a row: 0 holds the largest logit, the last whatever lies 37 or more below it in units of T (no mass) or
// the smallest.  fp32 subtraction and product are monotone, so a bin never holds a logit above one of an earlier bin.
struct SampleBins {
  float zmax, c;
  int last;
};
__device__ __forceinline__ SampleBins sample_bins(unsigned kmax, unsigned kmin, double invT, int bins) {
  const float zmax = sample_unkey(kmax);
  const double range = fmin(((double)zmax - (double)sample_unkey(kmin)) * invT, 37.0);
  return SampleBins{zmax, range > 0.0 ? (float)(bins * invT / range) : 0.f, bins - 1};
}
__device__ __forceinline__ int sample_bin(const SampleBins& b, float z) {
  const float x = (b.zmax - z) * b.c;
  return z == b.zmax ? 0 : (int)fminf(x, (float)b.last);
}

// One workgroup per row, any row: read again for every digit of the two selections.  What the kernels below do not take: rows with more
// codes around a cut than they hold (heavy ties).
template <typename T, int NT>
__device__ void sample_one_row(const SampleArgs& a, long row) {
  __shared__ unsigned long long hist_m[256];
  __shared__ unsigned hist_c[256];
  __shared__ unsigned long long part[(NT / 64)];
  __shared__ unsigned ties[(NT / 64)];
  __shared__ unsigned long long sh_m[3];
  __shared__ unsigned sh_c[3];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.V;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const SampleRow s = sample_row(a, row);

  // the largest logit and the lowest index that holds it
  unsigned long long best = 0;
  for (int i = tid; i < V; i += NT) {
    const unsigned long long c = (unsigned long long)sample_key(GroupNum<T>::get(z[i])) << 32 | (unsigned)~i;
    best = c > best ? c : best;
  }
  for (int m = 32; m > 0; m >>= 1) {
    const unsigned long long o = __shfl_xor(best, m, 64);
    best = o > best ? o : best;
  }
  if (lane == 0) part[w] = best;
  __syncthreads();
#pragma unroll 1
  for (int v = 0; v < (NT / 64); ++v) best = part[v] > best ? part[v] : best;
  __syncthreads();
  const unsigned kmax = (unsigned)(best >> 32);
  if (kmax <= kSampleKeyMasked) {
    if (tid == 0) sample_answer(a, row, -1, -INFINITY);
    return;
  }
  if (s.greedy) {
    if (tid == 0) sample_answer(a, row, (long)(unsigned)~(unsigned)best, 0.f);
    return;
  }
  const double zmax = (double)sample_unkey(kmax), scale = ldexp(1.0, a.F);
  auto mass = [&](unsigned key) { return sample_mass(sample_arg(key, kmax, zmax, s.invT), scale, 0.0); };

  // t, r: codes above t are kept, and the first r of those at t.  Top-k by counts, 8 bits at a time from the top.
  unsigned t = kSampleKeyMasked, r = 0;
  if (s.k < V) {
    unsigned prefix = 0, want = (unsigned)s.k;   // the want-th largest among the keys that share the prefix
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist_c[tid] = 0;
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < V; i += NT) {
        const unsigned key = sample_key(GroupNum<T>::get(z[i]));
        if (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist_c[(key >> shift) & 255], 1u);
      }
      __syncthreads();
      if (tid == 0) {
        unsigned above = 0;
        int d = 255;
        while (above + hist_c[d] < want) above += hist_c[d--];
        sh_c[0] = (unsigned)d;
        sh_c[1] = want - above;
      }
      __syncthreads();
      prefix |= sh_c[0] << shift;
      want = sh_c[1];
      __syncthreads();
    }
    if (prefix > kSampleKeyMasked) {   // (fewer than k codes are left otherwise: all of them are kept)
      t = prefix;
      r = want;
    }
  }
  // Top-p by mass among those: the lowest key whose codes have less than p of the mass before them
  if (s.p < 1.0) {
    unsigned prefix = 0;
    unsigned long long bound = 0, before = 0;
#pragma unroll 1
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist_m[tid] = 0;
      __syncthreads();
#pragma unroll 1
      for (int i = tid; i < V; i += NT) {
        const unsigned key = sample_key(GroupNum<T>::get(z[i]));
        if (key > t && (shift == 24 || key >> (shift + 8) == prefix >> (shift + 8))) {
          const unsigned long long q = mass(key);
          if (q) atomicAdd(&hist_m[(key >> shift) & 255], q);
        }
      }
      __syncthreads();
      if (tid == 0) {
        if (r && (shift == 24 || t >> (shift + 8) == prefix >> (shift + 8))) hist_m[(t >> shift) & 255] += r * mass(t);
        if (shift == 24) {
          unsigned long long total = 0;
  #pragma unroll 1
          for (int d = 0; d < 256; ++d) total += hist_m[d];
          sh_m[1] = sample_bound(s.p, total);
        }
        const unsigned long long lim = shift == 24 ? sh_m[1] : bound;
        unsigned long long run = before;
        int d = 255;
        while (run + hist_m[d] < lim) run += hist_m[d--];
        sh_m[0] = run;
        sh_c[0] = (unsigned)d;
      }
      __syncthreads();
      prefix |= sh_c[0] << shift;
      before = sh_m[0];
      if (shift == 24) bound = sh_m[1];
      __syncthreads();
    }
    const unsigned long long q = mass(prefix);   // > 0: the digit walk ends on a key that has mass
    const unsigned need = sample_ceil_div(bound - before, q);
    r = prefix == t && r < need ? r : need;
    t = prefix;
  }
  // mass of the kept codes, wave by wave: wave w owns a run of indexes, so that ties are counted and the draw walks in index order
  const int seg = ((V + (NT / 64) * 64 - 1) / ((NT / 64) * 64)) * 64;
  const int i0 = w * seg, i1 = i0 + seg < V ? i0 + seg : V;
  const unsigned long long qt = r ? sample_mass(sample_arg(t, kmax, zmax, s.invT), scale, s.m) : 0;
  auto kept = [&](unsigned key) { return key > t ? sample_mass(sample_arg(key, kmax, zmax, s.invT), scale, s.m) : 0ull; };
  unsigned long long sum = 0;
  unsigned tie = 0;
#pragma unroll 1
  for (int i = i0 + lane; i < i1; i += 64) {
    const unsigned key = sample_key(GroupNum<T>::get(z[i]));
    sum += kept(key);
    tie += key == t;
  }
  sum = sample_wave_sum(sum);
  tie = sample_wave_sum(tie);
  if (lane == 0) {
    part[w] = sum;
    ties[w] = tie;
  }
  __syncthreads();
  unsigned long long total = 0, my_before = 0;
  unsigned tie_before = 0, seen = 0;
#pragma unroll 1
  for (int v = 0; v < (NT / 64); ++v) {
    if (v == w) {
      my_before = total;
      tie_before = seen;
    }
    const unsigned left = r > seen ? r - seen : 0;
    total += part[v] + (ties[v] < left ? ties[v] : left) * qt;
    seen += ties[v];
  }
  // the lowest index at which the running mass passes u * total
  unsigned long long target = (unsigned long long)(s.u * (double)total);
  if (target >= total) target = total - 1;
  const unsigned left = r > tie_before ? r - tie_before : 0;
  const unsigned long long mine = sum + (tie < left ? tie : left) * qt;
  if (my_before <= target && target < my_before + mine) {
    unsigned long long run = my_before;
    unsigned tied = tie_before;
    for (int i = i0; i < i1; i += 64) {
      const unsigned key = i + lane < i1 ? sample_key(GroupNum<T>::get(z[i + lane])) : 0u;
      const unsigned long long at = __ballot(key == t && r > 0);
      const unsigned nth = tied + __builtin_popcountll(at & ((1ull << lane) - 1));
      unsigned long long q = kept(key);
      if (key == t && r > 0) q = nth < r ? qt : 0;
      const unsigned long long incl = run + sample_wave_scan(q);
      const unsigned long long hit = __ballot(incl > target);
      if (hit) {
        const int first = __builtin_ctzll(hit);
        if (lane == first)
          sample_answer(a, row, i + lane, (float)(sample_arg(key, kmax, zmax, s.invT) - log((double)total / scale)));
        break;
      }
      run = sample_lane(incl, 63);
      tied += __builtin_popcountll(at);
    }
  }
}

// One wave per row, V <= 64 R: the row stays in registers (lane l holds codes l R ... l R + R - 1), no barrier anywhere.
// Both cuts look at 64 bins of the row first (counts and masses by LDS atomics, scanned by the wave), then at the few codes of the one
// bin that the cut falls into, a lane each.  A bin of more than 64 codes (heavy ties) is searched bit by bit instead.
constexpr int kSampleRowWaves = 4;
struct SampleWaveLds {
  unsigned long long mass[64];
  unsigned count[64];
  unsigned long long m_mass[64];   // members of the bin in question
  unsigned m_key[64];
};

template <int R>
struct SampleWaveRow {
  unsigned key[R];
  unsigned long long q[R];

  // codes with bin(z) == b into the members' arrays; more than 64: -1
  __device__ int members(SampleWaveLds& s, const SampleBins& bins, unsigned b) const {
    const int lane = threadIdx.x & 63;
    int n = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool in = key[j] > kSampleKeyMasked && (unsigned)sample_bin(bins, sample_unkey(key[j])) == b;
      const unsigned long long at = __ballot(in);
      const int to = n + (int)__builtin_popcountll(at & ((1ull << lane) - 1));
      if (in && to < 64) {
        s.m_key[to] = key[j];
        s.m_mass[to] = q[j];
      }
      n += (int)__builtin_popcountll(at);
    }
    return n <= 64 ? n : -1;
  }
};

template <typename T, int R>
__global__ void __launch_bounds__(64 * kSampleRowWaves) sample_wave_kernel(SampleArgs a) {
  __shared__ SampleWaveLds lds[kSampleRowWaves];
  SampleWaveLds& s = lds[threadIdx.x >> 6];
  const int lane = threadIdx.x & 63, V = a.V;
  const double scale = ldexp(1.0, a.F);
  for (long row = (long)blockIdx.x * kSampleRowWaves + (threadIdx.x >> 6); row < a.n; row += (long)gridDim.x * kSampleRowWaves) {
    const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    const SampleRow set = sample_row(a, row);
    SampleWaveRow<R> w;
    unsigned hi = 0, lo = 0;   // lo: the smallest key that is not masked, complemented
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int i = lane * R + j;
      w.key[j] = i < V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
      hi = max(hi, w.key[j]);
      lo = max(lo, w.key[j] > kSampleKeyMasked ? ~w.key[j] : 0u);
    }
    const unsigned kmax = sample_wave_max(hi), kmin = ~sample_wave_max(lo);
    if (kmax <= kSampleKeyMasked) {
      if (lane == 0) sample_answer(a, row, -1, -INFINITY);
      continue;
    }
    if (set.greedy) {
      const int first = __builtin_ctzll(__ballot(hi == kmax));
      int at = 0;
#pragma unroll
      for (int j = R - 1; j >= 0; --j) at = w.key[j] == kmax ? j : at;
      if (lane == first) sample_answer(a, row, lane * R + at, 0.f);
      continue;
    }
    const double zmax = (double)sample_unkey(kmax);
    unsigned floored = 0;   // bit j: cut by min-p
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const double e = sample_exp(sample_arg(w.key[j], kmax, zmax, set.invT));
      w.q[j] = w.key[j] > kSampleKeyMasked ? sample_whole(e, scale) : 0ull;
      floored |= (e >= set.m ? 0u : 1u) << j;
    }
    unsigned t = kSampleKeyMasked, r = 0;
    const bool by_count = set.k < V, by_mass = set.p < 1.0;
    if (by_count || by_mass) {
      const SampleBins bins = sample_bins(kmax, kmin, set.invT, 64);
      s.mass[lane] = 0;
      s.count[lane] = 0;
      sample_wave_sync();
#pragma unroll
      for (int j = 0; j < R; ++j) {
        if (w.key[j] > kSampleKeyMasked) {
          const int b = sample_bin(bins, sample_unkey(w.key[j]));
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
      if (by_count && set.k < (int)sample_lane(c_run, 63)) {
        kb = __builtin_ctzll(__ballot(c_run >= (unsigned)set.k));
        const unsigned want = (unsigned)set.k - (sample_lane(c_run, kb) - sample_lane(c_in, kb));
        const unsigned long long above = sample_lane(m_run, kb) - sample_lane(m_in, kb);
        n_kb = w.members(s, bins, kb);
        sample_wave_sync();
        if (n_kb >= 0) {
          const unsigned mk = lane < n_kb ? s.m_key[lane] : 0u;
          const unsigned long long mq = lane < n_kb ? s.m_mass[lane] : 0ull;
          unsigned gt = 0, ge = 0;
          for (int i = 0; i < n_kb; ++i) {
            const unsigned o = sample_lane(mk, i);
            gt += o > mk;
            ge += o >= mk;
          }
          const int at = __builtin_ctzll(__ballot(lane < n_kb && gt < want && want <= ge));
          t = sample_lane(mk, at);
          r = want - sample_lane(gt, at);
          total = above + sample_wave_sum(mk > t ? mq : 0ull) + r * sample_lane(mq, at);
        } else {   // the largest t that at least k keys reach, a bit at a time
          unsigned key = 0;
          for (int b = 31; b >= 0; --b) {
            const unsigned c = key | 1u << b;
            unsigned n = 0;
#pragma unroll
            for (int j = 0; j < R; ++j) n += (unsigned)__builtin_popcountll(__ballot(w.key[j] >= c));
            if (n >= (unsigned)set.k) key = c;
          }
          t = key;
          unsigned n = 0;
          unsigned long long m = 0;
#pragma unroll
          for (int j = 0; j < R; ++j) {
            n += (unsigned)__builtin_popcountll(__ballot(w.key[j] > t));
            m += w.key[j] > t ? w.q[j] : 0ull;
          }
          r = (unsigned)set.k - n;
          total = sample_wave_sum(m) + r * sample_mass(sample_arg(t, kmax, zmax, set.invT), scale, 0.0);
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
          const unsigned mk = lane < n ? s.m_key[lane] : 0u;
          unsigned long long mq = lane < n ? s.m_mass[lane] : 0ull;
          if (mk <= t) mq = 0;
          unsigned long long gt = 0, ge = 0;
          for (int i = 0; i < n; ++i) {
            const unsigned o = sample_lane(mk, i);
            const unsigned long long m = sample_lane(mq, i);
            gt += o > mk ? m : 0ull;
            ge += o >= mk ? m : 0ull;
          }
          const unsigned long long hit = __ballot(mk > t && gt < need && need <= ge);
          if (hit) {   // (else it falls on the ties that top-k kept)
            const int at = __builtin_ctzll(hit);
            t = sample_lane(mk, at);
            r = sample_ceil_div(need - sample_lane(gt, at), sample_lane(mq, at));
          } else {
            r = min(r, sample_ceil_div(need - sample_wave_sum(mq), sample_mass(sample_arg(t, kmax, zmax, set.invT), scale, 0.0)));
          }
        } else {
          const unsigned long long at_t = r ? r * sample_mass(sample_arg(t, kmax, zmax, set.invT), scale, 0.0) : 0ull;
          unsigned key = 0;
          for (int b = 31; b >= 0; --b) {
            const unsigned c = key | 1u << b;
            unsigned long long m = 0;
#pragma unroll
            for (int j = 0; j < R; ++j) m += w.key[j] >= c && w.key[j] > t ? w.q[j] : 0ull;
            if (sample_wave_sum(m) + (t >= c ? at_t : 0ull) >= bound) key = c;
          }
          unsigned long long m = 0;
#pragma unroll
          for (int j = 0; j < R; ++j) m += w.key[j] > key && w.key[j] > t ? w.q[j] : 0ull;
          const unsigned rr = sample_ceil_div(bound - sample_wave_sum(m) - (t > key ? at_t : 0ull),
                                              sample_mass(sample_arg(key, kmax, zmax, set.invT), scale, 0.0));
          r = key == t ? min(r, rr) : rr;
          t = key;
        }
      }
    }
    // the draw: kept masses summed in index order
    unsigned ties = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) ties += w.key[j] == t;
    unsigned nth = 0;
    if (r) nth = sample_wave_scan(ties) - ties;
    unsigned long long sum = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const bool tie = w.key[j] == t;
      const bool kept = (w.key[j] > t || (tie && nth < r)) && !(floored >> j & 1);
      nth += tie;
      w.q[j] = kept ? w.q[j] : 0ull;
      sum += w.q[j];
    }
    const unsigned long long run = sample_wave_scan(sum), total = sample_lane(run, 63);
    unsigned long long target = (unsigned long long)(set.u * (double)total);
    if (target >= total) target = total - 1;
    const int first = __builtin_ctzll(__ballot(run > target));
    if (lane == first) {
      unsigned long long upto = run - sum;
      int at = 0;
      unsigned key = 0;
      bool found = false;
#pragma unroll
      for (int j = 0; j < R; ++j) {
        upto += w.q[j];
        if (!found && upto > target) {
          found = true;
          at = j;
          key = w.key[j];
        }
      }
      sample_answer(a, row, lane * R + at, (float)(sample_arg(key, kmax, zmax, set.invT) - log((double)total / scale)));
    }
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// Longer rows.  The same two looks, by workgroups: 1024 bins of the row (counts and masses), then the codes ("members") of the bins
// that the cuts fall into.  Where both cuts are on, what top-k keeps of its bin is not known before its members are looked at; the mass
// that top-p cuts at is then known only to within that bin's mass, and the members of all bins it can fall into are taken.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSampleBins = 1024;
constexpr unsigned kSampleFloored = 1u << 31;   // flag beside a member's index (< 2^24): cut by min-p

struct SampleCuts {
  int kb;                              // the bin that top-k cuts; kSampleBins: none
  unsigned want;                       // codes kept of it
  unsigned long long above, k_mass;    // mass before it, and of it
  int b0, b1;                          // bins that the last cut falls into; bins before b0 are kept whole; b0 == kSampleBins: no cut
  unsigned long long base;             // mass before b0
  unsigned long long bound;            // the mass that top-p cuts at, where top-k cuts nothing
};
__device__ __forceinline__ bool sample_is_member(const SampleCuts& c, int b) { return b >= c.b0 && (b <= c.b1 || b == c.kb); }

template <int NT>
struct SampleBlock {
  unsigned long long m[NT / 64];
  unsigned c[NT / 64];
};
// exclusive scan over the workgroup's threads of a mass and a count, and their totals.  Barriers: one before its reads, one behind.
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
  m_before = mi - m;
  c_before = ci - c;
  m_all = 0;
  c_all = 0;
#pragma unroll 4
  for (int v = 0; v < NT / 64; ++v) {
    m_before += v < w ? s.m[v] : 0;
    c_before += v < w ? s.c[v] : 0;
    m_all += s.m[v];
    c_all += s.c[v];
  }
  __syncthreads();
}

// the cuts' bins from the row's bins (LDS); every thread, result in `out` (LDS)
template <int NT>
__device__ __forceinline__ void sample_find_cuts(SampleBlock<NT>& blk, const unsigned* count, const unsigned long long* mass, const SampleRow& s,
                                                 int V, SampleCuts& out) {
  constexpr int PB = kSampleBins / NT;
  static_assert(PB >= 1, "a thread owns whole bins");
  const int b0 = threadIdx.x * PB;
  unsigned long long m = 0, m_before, m_all;
  unsigned c = 0, c_before, c_all;
  for (int j = 0; j < PB; ++j) {
    m += mass[b0 + j];
    c += count[b0 + j];
  }
  if (threadIdx.x == 0) {
    out.kb = out.b0 = out.b1 = kSampleBins;
    out.want = 0;
    out.above = out.k_mass = out.base = out.bound = 0;
  }
  sample_block_scan<NT>(blk, m, c, m_before, c_before, m_all, c_all);
  if (s.k < V && (unsigned)s.k < c_all) {
    unsigned long long mr = m_before;
    unsigned cr = c_before;
    for (int j = 0; j < PB; ++j) {
      const unsigned n = count[b0 + j];
      if (cr < (unsigned)s.k && (unsigned)s.k <= cr + n) {
        out.kb = out.b0 = out.b1 = b0 + j;
        out.want = (unsigned)s.k - cr;
        out.above = out.base = mr;
        out.k_mass = mass[b0 + j];
      }
      cr += n;
      mr += mass[b0 + j];
    }
  }
  __syncthreads();
  if (s.p < 1.0) {
    const bool cut = out.kb < kSampleBins;
    const unsigned long long lo = sample_bound(s.p, cut ? out.above : m_all), hi = sample_bound(s.p, cut ? out.above + out.k_mass : m_all);
    __syncthreads();
    unsigned long long mr = m_before;
    for (int j = 0; j < PB; ++j) {
      const unsigned long long n = mass[b0 + j];
      if (mr < lo && lo <= mr + n) {
        out.b0 = b0 + j;
        out.base = mr;
      }
      if (mr < hi && hi <= mr + n) out.b1 = b0 + j;
      mr += n;
    }
    if (!cut && threadIdx.x == 0) out.bound = lo;
    __syncthreads();
  }
}

// t and r from the members (LDS arrays of n; of any order): see the top of the file.  sh: scratch in LDS.
struct SampleFound {
  unsigned t, r;
  int hit;
};
template <int NT>
__device__ __forceinline__ void sample_resolve(SampleBlock<NT>& blk, SampleFound& sh, const SampleCuts& cut, const SampleBins& bins,
                                               const unsigned* m_key, const unsigned long long* m_mass, int n, double p, unsigned& t, unsigned& r) {
  t = kSampleKeyMasked;
  r = 0;
  unsigned long long total = 0, none;
  unsigned none_c, c_all;
  unsigned long long qt = 0;   // mass of one code at t
  if (cut.kb < kSampleBins) {
    for (int i = threadIdx.x; i < n; i += NT) {
      const unsigned key = m_key[i];
      if (sample_bin(bins, sample_unkey(key)) == cut.kb) {
        unsigned gt = 0, ge = 0;
#pragma unroll 2
        for (int o = 0; o < n; ++o) {
          const unsigned ko = m_key[o];
          const bool in = sample_bin(bins, sample_unkey(ko)) == cut.kb;
          gt += in && ko > key;
          ge += in && ko >= key;
        }
        if (gt < cut.want && cut.want <= ge) {   // (equal keys find the same)
          sh.t = key;
          sh.r = cut.want - gt;
          sh.hit = i;
        }
      }
    }
    __syncthreads();
    t = sh.t;
    r = sh.r;
    qt = m_mass[sh.hit];
    unsigned long long m = 0;
    for (int i = threadIdx.x; i < n; i += NT)
      if (m_key[i] > t && sample_bin(bins, sample_unkey(m_key[i])) == cut.kb) m += m_mass[i];
    sample_block_scan<NT>(blk, m, 0u, none, none_c, total, c_all);
    total += cut.above + r * qt;
  }
  if (p < 1.0) {
    const unsigned long long bound = cut.kb < kSampleBins ? sample_bound(p, total) : cut.bound;
    if (threadIdx.x == 0) sh.hit = -1;
    unsigned long long m = 0;
    for (int i = threadIdx.x; i < n; i += NT) m += m_key[i] > t ? m_mass[i] : 0ull;
    unsigned long long all;
    sample_block_scan<NT>(blk, m, 0u, none, none_c, all, c_all);
    for (int i = threadIdx.x; i < n; i += NT) {
      const unsigned key = m_key[i];
      if (key > t) {
        unsigned long long gt = cut.base, eq = 0;
#pragma unroll 2
        for (int o = 0; o < n; ++o) {
          const unsigned ko = m_key[o];
          const unsigned long long q = m_mass[o];
          gt += ko > key ? q : 0ull;
          eq += ko == key ? q : 0ull;
        }
        if (gt < bound && bound <= gt + eq) {
          sh.t = key;
          sh.r = sample_ceil_div(bound - gt, m_mass[i]);
          sh.hit = i;
        }
      }
    }
    __syncthreads();
    if (sh.hit >= 0) {
      t = sh.t;
      r = sh.r;
    } else {   // on the ties that top-k kept
      r = min(r, sample_ceil_div(bound - cut.base - all, qt));
    }
    __syncthreads();
  }
}

// The draw among the codes [w0, w0 + 64 STEPS) of every wave (w0: the wave's own first code), `run0` of mass and `tied0` codes at t before
// the first wave's: the wave that the target falls into walks them, 64 neighbouring codes per step.  `sum` and `at_t`: the wave's own
// mass above t and codes at t.
template <typename T, int NT, int STEPS>
__device__ __forceinline__ void sample_draw(const SampleArgs& a, long row, const T* z, int w0, unsigned kmax, double zmax, const SampleRow& set,
                                            double scale, unsigned t, unsigned r, unsigned long long qt, const SampleBlock<NT>& blk,
                                            unsigned long long sum, unsigned at_t, unsigned long long run0, unsigned tied0,
                                            unsigned long long target, unsigned long long total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  unsigned long long run = run0;
  unsigned seen = tied0;
#pragma unroll 1
  for (int v = 0; v < w; ++v) {
    run += blk.m[v] + min(blk.c[v], r > seen ? r - seen : 0u) * qt;
    seen += blk.c[v];
  }
  const unsigned long long here = sum + min(at_t, r > seen ? r - seen : 0u) * qt;
  if (run <= target && target < run + here) {
#pragma unroll 1
    for (int j = 0; j < STEPS; ++j) {
      const int i = w0 + j * 64 + lane;
      const unsigned key = i < a.V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
      const bool tie = r > 0 && key == t;
      const unsigned long long at = __ballot(tie);
      const unsigned nth = seen + __builtin_popcountll(at & ((1ull << lane) - 1));
      const double x = sample_arg(key, kmax, zmax, set.invT);
      const unsigned long long kept = key > t ? sample_mass(x, scale, set.m) : (tie && nth < r ? qt : 0ull);
      const unsigned long long incl = run + sample_wave_scan(kept);
      const unsigned long long hit = __ballot(incl > target);
      if (hit) {
        if (lane == (int)__builtin_ctzll(hit)) sample_answer(a, row, i, (float)(x - log((double)total / scale)));
        break;
      }
      run = sample_lane(incl, 63);
      seen += __builtin_popcountll(at);
    }
  }
}

// One workgroup per row, its keys in registers: wave w owns a run of 64 KPT codes, 64 neighbouring ones per step.
template <typename T, int NT, int KPT>
__global__ void __launch_bounds__(NT) sample_block_kernel(SampleArgs a) {
  constexpr int kMost = 1024;   // members; a row with more of them (heavy ties) goes through sample_one_row
  __shared__ unsigned long long mass[kSampleBins];
  __shared__ unsigned count[kSampleBins];
  __shared__ unsigned long long m_mass[kMost];
  __shared__ unsigned m_key[kMost];
  __shared__ SampleBlock<NT> blk;
  __shared__ SampleCuts cut;
  __shared__ SampleFound found;
  __shared__ unsigned range[2][NT / 64];
  __shared__ int n_members;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.V, w0 = w * 64 * KPT;
  const double scale = ldexp(1.0, a.F);
  for (long row = blockIdx.x; row < a.n; row += gridDim.x) {
    const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
    const SampleRow set = sample_row(a, row);
    unsigned key[KPT], hi = 0, lo = 0;
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
      const int i = w0 + j * 64 + lane;
      key[j] = i < V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
      hi = max(hi, key[j]);
      lo = max(lo, key[j] > kSampleKeyMasked ? ~key[j] : 0u);
    }
    hi = sample_wave_max(hi);
    lo = sample_wave_max(lo);
    if (lane == 0) {
      range[0][w] = hi;
      range[1][w] = lo;
    }
    for (int b = tid; b < kSampleBins; b += NT) {
      mass[b] = 0;
      count[b] = 0;
    }
    if (tid == 0) n_members = 0;
    __syncthreads();
#pragma unroll 4
    for (int v = 0; v < NT / 64; ++v) {
      hi = max(hi, range[0][v]);
      lo = max(lo, range[1][v]);
    }
    const unsigned kmax = hi, kmin = ~lo;
    if (kmax <= kSampleKeyMasked || set.greedy) {
      unsigned first = ~0u;
#pragma unroll
      for (int j = KPT - 1; j >= 0; --j)
        if (key[j] == kmax) first = w0 + j * 64 + lane;
      first = ~sample_wave_max(~first);
      __syncthreads();
      if (lane == 0) range[0][w] = first;
      __syncthreads();
      if (tid == 0) {
        for (int v = 1; v < NT / 64; ++v) first = min(first, range[0][v]);
        if (kmax <= kSampleKeyMasked) sample_answer(a, row, -1, -INFINITY);
        else sample_answer(a, row, (long)first, 0.f);
      }
      __syncthreads();
      continue;
    }
    const double zmax = (double)sample_unkey(kmax);
    auto mass_of = [&](unsigned k, double m) { return sample_mass(sample_arg(k, kmax, zmax, set.invT), scale, m); };
    unsigned t = kSampleKeyMasked, r = 0;
    const bool by_mass = set.p < 1.0;
    if (set.k < V || by_mass) {
      const SampleBins bins = sample_bins(kmax, kmin, set.invT, kSampleBins);
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        if (key[j] > kSampleKeyMasked) {
          const int b = sample_bin(bins, sample_unkey(key[j]));
          atomicAdd(&count[b], 1u);
          if (by_mass) {
            const unsigned long long q = mass_of(key[j], 0.0);
            if (q) atomicAdd(&mass[b], q);
          }
        }
        if (j & 1) __builtin_amdgcn_sched_barrier(0);   // (two exponentials at a time: sixteen of them side by side take registers)
      }
      __syncthreads();
      sample_find_cuts<NT>(blk, count, mass, set, V, cut);
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        if (key[j] > kSampleKeyMasked && sample_is_member(cut, sample_bin(bins, sample_unkey(key[j])))) {
          const int to = atomicAdd(&n_members, 1);
          if (to < kMost) m_key[to] = key[j];
        }
      }
      __syncthreads();
      const int n = n_members;
      if (n > kMost) {
        sample_one_row<T, NT>(a, row);
        __syncthreads();
        continue;
      }
      for (int i = tid; i < n; i += NT) m_mass[i] = mass_of(m_key[i], 0.0);
      __syncthreads();
      sample_resolve<NT>(blk, found, cut, bins, m_key, m_mass, n, set.p, t, r);
    }
    // kept masses, wave by wave
    unsigned at_t = 0;
    unsigned long long sum = 0;
#pragma unroll
    for (int j = 0; j < KPT; ++j) {
      at_t += key[j] == t && r > 0;
      if (key[j] > t) sum += mass_of(key[j], set.m);
      if (j & 1) __builtin_amdgcn_sched_barrier(0);
    }
    const unsigned long long qt = r ? mass_of(t, set.m) : 0ull;
    at_t = sample_wave_sum(at_t);
    sum = sample_wave_sum(sum);
    if (lane == 0) {
      blk.m[w] = sum;
      blk.c[w] = at_t;
    }
    __syncthreads();
    unsigned long long total = 0;
    unsigned seen = 0;
#pragma unroll 1
    for (int v = 0; v < NT / 64; ++v) {
      total += blk.m[v] + min(blk.c[v], r > seen ? r - seen : 0u) * qt;
      seen += blk.c[v];
    }
    unsigned long long target = (unsigned long long)(set.u * (double)total);
    if (target >= total) target = total - 1;
    sample_draw<T, NT, KPT>(a, row, z, w0, kmax, zmax, set, scale, t, r, qt, blk, sum, at_t, 0ull, 0u, target, total);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------------
// The longest rows, a workgroup per chunk of 16384 codes: (1) largest and smallest logit of every chunk, (2) its bins, summed over the
// chunks, (3) members, and the mass of what is kept whole in every chunk, (4) one workgroup per row: the cuts, the chunk that the draw
// falls into, and the code in it.  Three passes over the logits, of which the cache serves the later two; no atomics on floats, and
// nobody waits for another workgroup inside a kernel.
// ---------------------------------------------------------------------------------------------------------------------
constexpr int kSampleChunk = 16384, kSampleChunkThreads = 1024, kSampleChunkIpt = kSampleChunk / kSampleChunkThreads;
constexpr int kSampleMaxChunks = 1024;      // V <= 2^24
constexpr int kSampleMembers = 2048;        // of a row; with more (heavy ties) the row goes through sample_one_row

struct SampleLong {
  long row0;                                // first row of the batch
  int chunks;
  unsigned long long* best;                 // [row][chunk] largest key << 32 | ~lowest index that holds it
  unsigned* least;                          // [row][chunk] smallest key that is not masked, complemented
  unsigned long long* mass;                 // [row][chunk][bin]
  unsigned* count;
  unsigned long long* row_mass;             // [row][bin]
  unsigned* row_count;
  SampleCuts* cuts;                         // [row]
  unsigned long long* chunk_mass;           // [row][chunk] of codes kept whole
  int* n_members;                           // [row]
  unsigned long long* m_mass;               // [row][kSampleMembers]
  unsigned* m_key;
  unsigned* m_idx;                          // index, kSampleFloored
};

struct SampleRange {
  unsigned kmax, kmin, first;               // first: lowest index of kmax
};
// the row's range from its chunks'; every thread, with scratch in LDS
template <int NT>
__device__ __forceinline__ SampleRange sample_range(const SampleLong& l, long r, unsigned long long* sh_best, unsigned* sh_least) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  unsigned long long best = 0;
  unsigned least = 0;
  for (int c = threadIdx.x; c < l.chunks; c += NT) {
    const unsigned long long b = l.best[r * l.chunks + c];
    best = b > best ? b : best;
    least = max(least, l.least[r * l.chunks + c]);
  }
  const unsigned key = sample_wave_max((unsigned)(best >> 32));
  const unsigned at = sample_wave_max((unsigned)(best >> 32) == key ? (unsigned)best : 0u);
  least = sample_wave_max(least);
  if (lane == 0) {
    sh_best[w] = (unsigned long long)key << 32 | at;
    sh_least[w] = least;
  }
  __syncthreads();
  best = 0;
#pragma unroll 4
  for (int v = 0; v < NT / 64; ++v) {
    best = sh_best[v] > best ? sh_best[v] : best;
    least = max(least, sh_least[v]);
  }
  __syncthreads();
  return SampleRange{(unsigned)(best >> 32), ~least, ~(unsigned)best};
}

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_range_kernel(SampleArgs a, SampleLong l) {
  __shared__ unsigned long long sh_best[kSampleChunkThreads / 64];
  __shared__ unsigned sh_least[kSampleChunkThreads / 64];
  const long r = blockIdx.x / l.chunks;
  const int c = blockIdx.x - (int)(r * l.chunks), i0 = c * kSampleChunk, tid = threadIdx.x;
  const T* z = reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride;
  unsigned key[kSampleChunkIpt], hi = 0, least = 0;
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    const int i = i0 + j * kSampleChunkThreads + tid;
    key[j] = i < a.V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
    hi = max(hi, key[j]);
    least = max(least, key[j] > kSampleKeyMasked ? ~key[j] : 0u);
  }
  unsigned at = 0;
#pragma unroll
  for (int j = kSampleChunkIpt - 1; j >= 0; --j)
    if (key[j] == hi) at = ~(unsigned)(i0 + j * kSampleChunkThreads + tid);
  const unsigned top = sample_wave_max(hi);
  at = sample_wave_max(hi == top ? at : 0u);
  least = sample_wave_max(least);
  if ((tid & 63) == 0) {
    sh_best[tid >> 6] = (unsigned long long)top << 32 | at;
    sh_least[tid >> 6] = least;
  }
  __syncthreads();
  if (tid == 0) {
    unsigned long long best = 0;
    for (int v = 0; v < kSampleChunkThreads / 64; ++v) {
      best = sh_best[v] > best ? sh_best[v] : best;
      least = max(least, sh_least[v]);
    }
    l.best[r * l.chunks + c] = best;
    l.least[r * l.chunks + c] = least;
    if (c == 0) l.n_members[r] = 0;
  }
}

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_bins_kernel(SampleArgs a, SampleLong l) {
  __shared__ unsigned long long mass[kSampleBins];
  __shared__ unsigned count[kSampleBins];
  __shared__ unsigned long long sh_best[kSampleChunkThreads / 64];
  __shared__ unsigned sh_least[kSampleChunkThreads / 64];
  static_assert(kSampleBins == kSampleChunkThreads, "a thread owns a bin");
  const long r = blockIdx.x / l.chunks;
  const int c = blockIdx.x - (int)(r * l.chunks), i0 = c * kSampleChunk, tid = threadIdx.x;
  const SampleRow set = sample_row(a, l.row0 + r);
  const bool by_mass = set.p < 1.0;
  if (set.greedy || !(set.k < a.V || by_mass)) return;
  const T* z = reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride;
  unsigned key[kSampleChunkIpt];
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    const int i = i0 + j * kSampleChunkThreads + tid;
    key[j] = i < a.V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
  }
  mass[tid] = 0;
  count[tid] = 0;
  const SampleRange g = sample_range<kSampleChunkThreads>(l, r, sh_best, sh_least);   // (its barriers: the bins are cleared)
  if (g.kmax <= kSampleKeyMasked) return;
  const double zmax = (double)sample_unkey(g.kmax), scale = ldexp(1.0, a.F);
  const SampleBins bins = sample_bins(g.kmax, g.kmin, set.invT, kSampleBins);
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    if (key[j] > kSampleKeyMasked) {
      const int b = sample_bin(bins, sample_unkey(key[j]));
      atomicAdd(&count[b], 1u);
      if (by_mass) {
        const unsigned long long q = sample_mass(sample_arg(key[j], g.kmax, zmax, set.invT), scale, 0.0);
        if (q) atomicAdd(&mass[b], q);
      }
    }
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
  }
  __syncthreads();
  const size_t o = ((size_t)r * l.chunks + c) * kSampleBins + tid;
  l.mass[o] = mass[tid];
  l.count[o] = count[tid];
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

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_members_kernel(SampleArgs a, SampleLong l) {
  constexpr int NT = kSampleChunkThreads;
  __shared__ unsigned long long mass[kSampleBins];
  __shared__ unsigned count[kSampleBins];
  __shared__ unsigned long long sh_best[NT / 64];
  __shared__ unsigned sh_least[NT / 64];
  __shared__ SampleBlock<NT> blk;
  __shared__ SampleCuts cut;
  __shared__ unsigned long long m_mass[kSampleMembers];
  __shared__ unsigned m_key[kSampleMembers], m_idx[kSampleMembers];
  __shared__ int n_here, first_here;
  const long r = blockIdx.x / l.chunks;
  const int c = blockIdx.x - (int)(r * l.chunks), i0 = c * kSampleChunk, tid = threadIdx.x;
  const SampleRow set = sample_row(a, l.row0 + r);
  if (set.greedy) return;
  const T* z = reinterpret_cast<const T*>(a.logits) + (l.row0 + r) * a.stride;
  unsigned key[kSampleChunkIpt];
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    const int i = i0 + j * NT + tid;
    key[j] = i < a.V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
  }
  const bool any = set.k < a.V || set.p < 1.0;
  if (any) {
    mass[tid] = l.row_mass[r * kSampleBins + tid];
    count[tid] = l.row_count[r * kSampleBins + tid];
  }
  if (tid == 0) {
    n_here = 0;
    cut.kb = cut.b0 = cut.b1 = kSampleBins;
  }
  const SampleRange g = sample_range<NT>(l, r, sh_best, sh_least);
  if (g.kmax <= kSampleKeyMasked) return;
  const double zmax = (double)sample_unkey(g.kmax), scale = ldexp(1.0, a.F);
  const SampleBins bins = sample_bins(g.kmax, g.kmin, set.invT, kSampleBins);
  if (any) sample_find_cuts<NT>(blk, count, mass, set, a.V, cut);
  unsigned long long sum = 0;
#pragma unroll
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    if (key[j] > kSampleKeyMasked) {
      const int b = sample_bin(bins, sample_unkey(key[j]));
      const bool member = sample_is_member(cut, b);
      if (b < cut.b0 || member) {
        const double e = sample_exp(sample_arg(key[j], g.kmax, zmax, set.invT));
        const unsigned long long q = sample_whole(e, scale);
        if (member) {
          const int to = atomicAdd(&n_here, 1);
          if (to < kSampleMembers) {
            m_key[to] = key[j];
            m_mass[to] = q;
            m_idx[to] = (unsigned)(i0 + j * NT + tid) | (e >= set.m ? 0u : kSampleFloored);
          }
        } else {
          sum += e >= set.m ? q : 0ull;
        }
      }
    }
    if (j & 1) __builtin_amdgcn_sched_barrier(0);
  }
  unsigned long long before, all;
  unsigned none, none_all;
  sample_block_scan<NT>(blk, sum, 0u, before, none, all, none_all);   // (its barriers: the members are all there)
  const int n = n_here;
  if (tid == 0) {
    l.chunk_mass[r * l.chunks + c] = all;
    if (c == 0) l.cuts[r] = cut;
    if (n) first_here = atomicAdd(&l.n_members[r], n);
  }
  __syncthreads();
  for (int i = tid; i < min(n, kSampleMembers); i += NT) {
    const int to = first_here + i;
    if (to < kSampleMembers) {
      l.m_key[r * kSampleMembers + to] = m_key[i];
      l.m_mass[r * kSampleMembers + to] = m_mass[i];
      l.m_idx[r * kSampleMembers + to] = m_idx[i];
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kSampleChunkThreads) sample_finish_kernel(SampleArgs a, SampleLong l) {
  constexpr int NT = kSampleChunkThreads;
  __shared__ unsigned long long sh_best[NT / 64];
  __shared__ unsigned sh_least[NT / 64];
  __shared__ SampleBlock<NT> blk;
  __shared__ SampleCuts cut;
  __shared__ SampleFound found;
  __shared__ unsigned long long m_mass[kSampleMembers];
  __shared__ unsigned m_key[kSampleMembers], m_idx[kSampleMembers];
  __shared__ unsigned long long chunk[kSampleMaxChunks];
  __shared__ int sh_chunk;
  __shared__ unsigned long long sh_before;
  const long r = blockIdx.x, row = l.row0 + r;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const SampleRow set = sample_row(a, row);
  const SampleRange g = sample_range<NT>(l, r, sh_best, sh_least);
  if (g.kmax <= kSampleKeyMasked || set.greedy) {
    if (tid == 0) {
      if (set.greedy && g.kmax > kSampleKeyMasked) sample_answer(a, row, (long)g.first, 0.f);
      else sample_answer(a, row, -1, -INFINITY);
    }
    return;
  }
  const int n = l.n_members[r];
  if (n > kSampleMembers) {
    sample_one_row<T, NT>(a, row);
    return;
  }
  const double zmax = (double)sample_unkey(g.kmax), scale = ldexp(1.0, a.F);
  const SampleBins bins = sample_bins(g.kmax, g.kmin, set.invT, kSampleBins);
  if (tid == 0) cut = l.cuts[r];
  for (int i = tid; i < n; i += NT) {
    m_key[i] = l.m_key[r * kSampleMembers + i];
    m_mass[i] = l.m_mass[r * kSampleMembers + i];
    m_idx[i] = l.m_idx[r * kSampleMembers + i];
  }
  chunk[tid] = tid < l.chunks ? l.chunk_mass[r * l.chunks + tid] : 0ull;
  __syncthreads();
  unsigned t = kSampleKeyMasked, t_codes = 0;
  if (n) sample_resolve<NT>(blk, found, cut, bins, m_key, m_mass, n, set.p, t, t_codes);
  const unsigned ties = t_codes;
  // kept members into their chunks
  for (int i = tid; i < n; i += NT) {
    const unsigned key = m_key[i], idx = m_idx[i] & ~kSampleFloored;
    bool kept = key > t;
    if (key == t) {
      unsigned nth = 0;
      for (int o = 0; o < n; ++o) nth += m_key[o] == t && (m_idx[o] & ~kSampleFloored) < idx;
      kept = nth < ties;
    }
    if (kept && !(m_idx[i] & kSampleFloored)) atomicAdd(&chunk[idx / kSampleChunk], m_mass[i]);
  }
  __syncthreads();
  unsigned long long before, total;
  unsigned none, none_all;
  const unsigned long long mine = chunk[tid];
  sample_block_scan<NT>(blk, mine, 0u, before, none, total, none_all);
  unsigned long long target = (unsigned long long)(set.u * (double)total);
  if (target >= total) target = total - 1;
  if (before <= target && target < before + mine) {
    sh_chunk = tid;
    sh_before = before;
  }
  __syncthreads();
  const int c = sh_chunk, i0 = c * kSampleChunk;
  const unsigned long long run0 = sh_before;
  // ... and in that chunk: wave w walks codes [i0 + w 1024, + 1024)
  unsigned earlier = 0;   // ties in earlier chunks
  if (ties)
    for (int i = tid; i < n; i += NT) earlier += m_key[i] == t && (m_idx[i] & ~kSampleFloored) < (unsigned)i0;
  unsigned long long none_m, none_m_all;
  unsigned tied0;
  sample_block_scan<NT>(blk, 0ull, earlier, none_m, none, none_m_all, tied0);
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const int w0 = i0 + w * 64 * kSampleChunkIpt;
  auto key_at = [&](int j) {
    const int i = w0 + j * 64 + lane;
    return i < a.V ? sample_key(GroupNum<T>::get(z[i])) : kSampleKeyMasked;
  };
  auto mass_of = [&](unsigned key) { return sample_mass(sample_arg(key, g.kmax, zmax, set.invT), scale, set.m); };
  const unsigned long long qt = ties ? mass_of(t) : 0ull;
  unsigned long long sum = 0;
  unsigned at_t = 0;
#pragma unroll 4
  for (int j = 0; j < kSampleChunkIpt; ++j) {
    const unsigned key = key_at(j);
    sum += key > t ? mass_of(key) : 0ull;
    at_t += key == t && ties > 0;
  }
  sum = sample_wave_sum(sum);
  at_t = sample_wave_sum(at_t);
  if (lane == 0) {
    blk.m[w] = sum;
    blk.c[w] = at_t;
  }
  __syncthreads();
  sample_draw<T, NT, kSampleChunkIpt>(a, row, z, w0, g.kmax, zmax, set, scale, t, ties, qt, blk, sum, at_t, run0, tied0, target, total);
}

}  // namespace qinco
