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
// e = exp(x) as a whole number of 2^-F (scale = 2^F <= 2^51: the sum with 2^52 rounds it to one, ties to even)
__device__ __forceinline__ unsigned long long sample_whole(double e, double scale) {
  return (unsigned long long)__double_as_longlong(fma(e, scale, 0x1p52)) & ((1ull << 52) - 1);
}
// ... zero for what min-p cuts
__device__ __forceinline__ unsigned long long sample_mass(double x, double scale, double m) {
  const double e = exp(x);
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
    const unsigned need = sample_ceil_div(bound - before, q);
    r = prefix == t && r < need ? r : need;
    t = prefix;
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
      run = sample_lane(incl, 63);
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
      const double e = exp(sample_arg(w.key[j], kmax, zmax, set.invT));
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

}  // namespace qinco
