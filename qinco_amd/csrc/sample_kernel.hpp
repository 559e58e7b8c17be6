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

constexpr int kSampleThreads = 1024, kSampleWaves = kSampleThreads / 64;
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
// mass as a whole number of 2^-F; zero for what min-p cuts
__device__ __forceinline__ unsigned long long sample_mass(double x, double scale, double m) {
  const double e = exp(x);
  return e >= m ? (unsigned long long)(e * scale + 0.5) : 0ull;
}

// smallest whole number that is at least p * total: "mass before < p * total" is "mass before < this"
__device__ __forceinline__ unsigned long long sample_bound(double p, unsigned long long total) {
  const double b = ceil(p * (double)total);
  const unsigned long long v = (unsigned long long)b;
  return v < 1 ? 1 : (v > total ? total : v);
}

template <typename T>
__device__ __forceinline__ T sample_wave_sum(T v) {
  for (int m = 32; m > 0; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}
template <typename T>
__device__ __forceinline__ T sample_wave_scan(T v) {   // inclusive
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < 64; d <<= 1) {
    const T o = __shfl_up(v, d, 64);
    if (lane >= d) v += o;
  }
  return v;
}

// One workgroup per row, any V: the row is read again for every digit of the two selections (from L2 behind the first time).
template <typename T>
__device__ void sample_one_row(const SampleArgs& a, long row) {
  __shared__ unsigned long long hist_m[256];
  __shared__ unsigned hist_c[256];
  __shared__ unsigned long long part[kSampleWaves];
  __shared__ unsigned ties[kSampleWaves];
  __shared__ unsigned long long sh_m[3];
  __shared__ unsigned sh_c[3];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, V = a.V;
  const T* z = reinterpret_cast<const T*>(a.logits) + row * a.stride;
  const SampleRow s = sample_row(a, row);

  // the largest logit and the lowest index that holds it
  unsigned long long best = 0;
  for (int i = tid; i < V; i += kSampleThreads) {
    const unsigned long long c = (unsigned long long)sample_key(GroupNum<T>::get(z[i])) << 32 | (unsigned)~i;
    best = c > best ? c : best;
  }
  for (int m = 32; m > 0; m >>= 1) {
    const unsigned long long o = __shfl_xor(best, m, 64);
    best = o > best ? o : best;
  }
  if (lane == 0) part[w] = best;
  __syncthreads();
  for (int v = 0; v < kSampleWaves; ++v) best = part[v] > best ? part[v] : best;
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
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist_c[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kSampleThreads) {
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
    for (int shift = 24; shift >= 0; shift -= 8) {
      if (tid < 256) hist_m[tid] = 0;
      __syncthreads();
      for (int i = tid; i < V; i += kSampleThreads) {
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
    const unsigned long long need = (bound - before + q - 1) / q;
    if (prefix == t) r = need < r ? (unsigned)need : r;
    else r = need < (unsigned)V ? (unsigned)need : (unsigned)V, t = prefix;
  }
  // mass of the kept codes, wave by wave: wave w owns a run of indexes, so that ties are counted and the draw walks in index order
  const int seg = ((V + kSampleWaves * 64 - 1) / (kSampleWaves * 64)) * 64;
  const int i0 = w * seg, i1 = i0 + seg < V ? i0 + seg : V;
  const unsigned long long qt = r ? sample_mass(sample_arg(t, kmax, zmax, s.invT), scale, s.m) : 0;
  auto kept = [&](unsigned key) { return key > t ? sample_mass(sample_arg(key, kmax, zmax, s.invT), scale, s.m) : 0ull; };
  unsigned long long sum = 0;
  unsigned tie = 0;
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
  for (int v = 0; v < kSampleWaves; ++v) {
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
      run = __shfl(incl, 63, 64);
      tied += __builtin_popcountll(at);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kSampleThreads) sample_row_kernel(SampleArgs a) {
  for (long row = blockIdx.x; row < a.n; row += gridDim.x) {
    sample_one_row<T>(a, row);
    __syncthreads();
  }
}

}  // namespace qinco
