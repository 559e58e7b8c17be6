// Rows grouped by inverted list (the router's dispatch): n rows with k list ids each -> the n k entries sorted by list, stably, and the
// rows carried into that order and back with weights.  The ids are the IVF column of a code matrix (k = 1: filling an index,
// reference qinco/search/search_utils.py:121-162) or the k nearest centroids of qinco_knn_search (multi-probe).
//
// SORT.  key_i = list of entry i; order = stable sort of the entries by key, a radix sort by digits of at most 11 bits, lowest digit
// first.  Every pass is stable and free of atomics whose order shows: a tile of entries counts its digits (histogram), the counts are
// summed down the tiles (scan), and every tile ranks its entries again, orders them by digit in LDS and writes them out in runs (scatter).
// The rank of an entry = the entries of the same digit before it: inside a wave by ballots over the digit's bits, across waves by a table
// in LDS.  `place` is the passes' permutations one after the other: each pass notes where it put every entry next to where it found it
// (neighbouring stores), and the last kernel follows the notes (reads that the cache serves) -- a 4-byte store to a random place costs
// a whole sector.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qinco {

constexpr int kGroupThreads = 512, kGroupWaves = kGroupThreads / 64;
constexpr int kGroupIpt = 8;                              // entries per thread of the one-workgroup sort
constexpr int kGroupTile = kGroupThreads * kGroupIpt;     // ... its most entries
constexpr int kGroupMaxBits = 11, kGroupMaxBins = 1 << kGroupMaxBits;
constexpr unsigned kGroupNone = 0xFFFFFFFFu;              // key of an entry without a list
constexpr int kGroupSmallOffsets = 4096;                  // lists up to which the one-workgroup kernel writes the offsets itself

struct GroupKeys {
  const void* lists;   // (n, k) of code_dtype, rows `stride` elements apart
  int code_dtype;      // QINCO_CODE_*
  long stride;
  unsigned k, N, E;    // N = n k entries
};

__device__ __forceinline__ unsigned group_key(const GroupKeys& g, unsigned i, bool& bad) {
  const unsigned row = g.k == 1 ? i : i / g.k;
  const long o = (long)row * g.stride + (i - row * g.k);
  long v;
  if (g.code_dtype == 0) v = (long)reinterpret_cast<const long long*>(g.lists)[o];
  else if (g.code_dtype == 1) v = reinterpret_cast<const int*>(g.lists)[o];
  else v = reinterpret_cast<const unsigned char*>(g.lists)[o];
  bad = v >= (long)g.E;
  return (v < 0 || bad) ? kGroupNone : (unsigned)v;
}

struct GroupPass {
  GroupKeys in;                          // first pass: the lists
  const unsigned long long* pair_in;     // later passes: key << 32 | entry as the pass before left them, `*total` of them
  unsigned long long* pair_out;          // ... and for the pass behind this one
  int* order;                            // last pass: entries in slot order
  unsigned* key_out;                     // last of several passes: keys in slot order
  int* place;                            // first pass: where each entry went, -1 without a list
  int* went;                             // later passes: where each pair went
  int* offsets;                          // written by a sort of one pass (E + 1), else null
  unsigned* counts;                      // [tile][bin], after the scan: entries of that bin in earlier tiles
  unsigned* totals;                      // [bin]
  unsigned* start;                       // last of several passes: first slot of each bin, and behind the last one (bins + 1)
  unsigned* total;                       // entries that have a list
  int* bad;                              // nullable: set to 1 if an id is >= E
  int shift, bits, first, last;
  int tiles;                             // few: counts are as the histogram left them, every workgroup sums them itself; 0: scanned
};

// one wave's counter of a digit in LDS: read and bumped by lanes of the same wave, whose LDS accesses execute in order
__device__ __forceinline__ unsigned group_seen(const unsigned short& c) { return __hip_atomic_load(&c, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }
__device__ __forceinline__ void group_bump(unsigned short& c, unsigned v) { __hip_atomic_store(&c, (unsigned short)v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }

// the lanes whose digit d (of up to BITS bits) is this lane's, by one ballot per bit: where the bit is set the ballot, else its complement
template <int BITS>
__device__ __forceinline__ unsigned long long group_match(unsigned d, bool valid) {
  const unsigned long long v = __ballot(valid);
  unsigned lo = (unsigned)v, hi = (unsigned)(v >> 32);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const unsigned long long set = __ballot(d >> b & 1);
    const unsigned mine = (unsigned)((int)(d << (31 - b)) >> 31);   // all ones where the bit is set
    lo &= ~((unsigned)set ^ mine);
    hi &= ~((unsigned)(set >> 32) ^ mine);
  }
  return (unsigned long long)hi << 32 | lo;
}

// ranks of a wave's entries among the wave's own of the same digit; `seen` (LDS, of the wave) counts on
template <int BITS, int IPT, typename Key>
__device__ __forceinline__ void group_rank(unsigned short* seen, Key key_of, int shift, unsigned mask, unsigned (&rank)[IPT], int rounds) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    rank[r] = 0;
    if (r < rounds) {
      const unsigned key = key_of(r);
      const bool valid = key != kGroupNone;
      const unsigned d = (key >> shift) & mask;
      const unsigned long long m = group_match<BITS>(d, valid);
      const unsigned below = __builtin_popcountll(m & ((1ull << lane) - 1));
      if (valid) {
        const unsigned n = group_seen(seen[d]);
        rank[r] = n + below;
        if (below == 0) group_bump(seen[d], n + __builtin_popcountll(m));
      }
    }
  }
}

template <int IPT>
__global__ void __launch_bounds__(kGroupThreads) group_hist_kernel(GroupPass a) {
  __shared__ unsigned hist[kGroupMaxBins];
  const int bins = 1 << a.bits;
  for (int b = threadIdx.x; b < bins; b += kGroupThreads) hist[b] = 0;
  const unsigned N = a.first ? a.in.N : *a.total;
  const unsigned mask = bins - 1;
  unsigned key[IPT];
  bool any_bad = false;
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const unsigned i = blockIdx.x * (unsigned)(kGroupThreads * IPT) + r * kGroupThreads + threadIdx.x;
    key[r] = kGroupNone;
    if (i < N) {
      bool bad = false;
      key[r] = a.first ? group_key(a.in, i, bad) : (unsigned)(a.pair_in[i] >> 32);
      any_bad |= bad;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < IPT; ++r)
    if (key[r] != kGroupNone) atomicAdd(&hist[(key[r] >> a.shift) & mask], 1u);
  if (any_bad && a.bad) *a.bad = 1;
  __syncthreads();
  for (int b = threadIdx.x; b < bins; b += kGroupThreads) a.counts[(size_t)blockIdx.x * bins + b] = hist[b];
}

// counts[tile][bin] -> entries of the bin in earlier tiles; totals[bin].  A workgroup owns 64 bins, its 16 waves a run of tiles each,
// held in registers up to 16 of them.
__global__ void __launch_bounds__(1024) group_scan_kernel(unsigned* counts, unsigned* totals, int tiles, int bins) {
  __shared__ unsigned part[16][64];
  constexpr int HELD = 16;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int bin = blockIdx.x * 64 + lane;
  const int per = (tiles + 15) / 16;
  const int t0 = w * per, t1 = t0 + per < tiles ? t0 + per : tiles;
  unsigned held[HELD], sum = 0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) held[j] = bin < bins && t0 + j < t1 ? counts[(size_t)(t0 + j) * bins + bin] : 0;
#pragma unroll
  for (int j = 0; j < HELD; ++j) sum += held[j];
  if (bin < bins)
    for (int t = t0 + HELD; t < t1; ++t) sum += counts[(size_t)t * bins + bin];
  part[w][lane] = sum;
  __syncthreads();
  unsigned run = 0, all = 0;
#pragma unroll
  for (int v = 0; v < 16; ++v) {
    const unsigned p = part[v][lane];
    run += v < w ? p : 0;
    all += p;
  }
  if (bin < bins) {
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
      if (t0 + j < t1) counts[(size_t)(t0 + j) * bins + bin] = run;
      run += held[j];
    }
    for (int t = t0 + HELD; t < t1; ++t) {
      const size_t o = (size_t)t * bins + bin;
      const unsigned c = counts[o];
      counts[o] = run;
      run += c;
    }
    if (w == 0) totals[bin] = all;
  }
}

// exclusive scan of v over the workgroup's threads; *all = the sum.  Ends with a barrier behind its last read of tmp.
__device__ __forceinline__ unsigned group_block_scan(unsigned v, unsigned* tmp, unsigned* all) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  unsigned s = v;
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned o = __shfl_up(s, d, 64);
    if (lane >= d) s += o;
  }
  if (lane == 63) tmp[w] = s;
  __syncthreads();
  unsigned before = 0, sum = 0;
  for (int i = 0; i < kGroupWaves; ++i) {
    const unsigned t = tmp[i];
    before += i < w ? t : 0;
    sum += t;
  }
  __syncthreads();
  *all = sum;
  return before + s - v;
}

template <int IPT>
__global__ void __launch_bounds__(kGroupThreads) group_scatter_kernel(GroupPass a) {
  constexpr int TILE = kGroupThreads * IPT, BPT = kGroupMaxBins / kGroupThreads;
  __shared__ unsigned long long tile[TILE];                      // the tile's pairs by digit
  __shared__ unsigned short whist[kGroupWaves][kGroupMaxBins];   // entries of a digit in the wave so far, then in the tile before the wave's
  __shared__ unsigned base[kGroupMaxBins];                       // first slot of the tile's entries of a digit, less their place in the tile
  __shared__ unsigned tmp[kGroupWaves];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int bins = 1 << a.bits;
  const unsigned mask = bins - 1;
  const unsigned N = a.first ? a.in.N : *a.total;
  const unsigned tile0 = blockIdx.x * (unsigned)TILE;
  unsigned long long pair[IPT];
  unsigned rank[IPT];
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const unsigned i = tile0 + w * (64 * IPT) + r * 64 + lane;
    pair[r] = ~0ull;
    if (i < N) {
      if (a.first) {
        bool bad;
        pair[r] = (unsigned long long)group_key(a.in, i, bad) << 32 | i;
      } else {
        pair[r] = a.pair_in[i];
      }
    }
  }
  // thread -> neighbouring bins (1 .. 4)
  const int bpt = (bins + kGroupThreads - 1) / kGroupThreads;
  unsigned mine[BPT], earlier[BPT], s = 0;
#pragma unroll
  for (int j = 0; j < BPT; ++j) {
    const int b = tid * bpt + j;
    const bool in = j < bpt && b < bins;
    mine[j] = earlier[j] = 0;
    if (a.tiles) {
      if (in) {
#pragma unroll 8
        for (int t = 0; t < a.tiles; ++t) {
          const unsigned c = a.counts[(size_t)t * bins + b];
          mine[j] += c;
          earlier[j] += t < (int)blockIdx.x ? c : 0;
        }
      }
    } else if (in) {
      mine[j] = a.totals[b];
      earlier[j] = a.counts[(size_t)blockIdx.x * bins + b];
    }
    s += mine[j];
  }
  for (int b = tid * 2; b < bins; b += kGroupThreads * 2)   // (two 16-bit counters per store; of one bin there are two all the same)
    for (int v = 0; v < kGroupWaves; ++v) *reinterpret_cast<unsigned*>(&whist[v][b]) = 0;
  unsigned all;
  unsigned start = group_block_scan(s, tmp, &all);   // (its barriers also stand between the clearing of whist and its use)
  auto key_of = [&](int r) { return (unsigned)(pair[r] >> 32); };
  if (a.bits <= 8) group_rank<8>(whist[w], key_of, a.shift, mask, rank, IPT);
  else group_rank<kGroupMaxBits>(whist[w], key_of, a.shift, mask, rank, IPT);
  __syncthreads();
  // counts per wave -> places in the tile
  unsigned here[BPT], h = 0;
#pragma unroll
  for (int j = 0; j < BPT; ++j) {
    const int b = tid * bpt + j;
    here[j] = 0;
    if (j < bpt && b < bins)
      for (int v = 0; v < kGroupWaves; ++v) here[j] += whist[v][b];
    h += here[j];
  }
  unsigned in_tile;
  unsigned at = group_block_scan(h, tmp, &in_tile);
#pragma unroll
  for (int j = 0; j < BPT; ++j) {
    const int b = tid * bpt + j;
    if (j < bpt && b < bins) {
      if (blockIdx.x == 0) {
        if (a.offsets && (unsigned)b < a.in.E) a.offsets[b] = (int)start;
        if (a.last && a.start) a.start[b] = start;
      }
      base[b] = start + earlier[j] - at;
      unsigned run = at;
      for (int v = 0; v < kGroupWaves; ++v) {
        const unsigned c = whist[v][b];
        whist[v][b] = (unsigned short)run;
        run += c;
      }
      start += mine[j];
      at += here[j];
    }
  }
  if (blockIdx.x == 0 && tid == 0) {
    if (a.offsets) a.offsets[a.in.E] = (int)all;
    if (a.last && a.start) a.start[bins] = all;
    if (a.first) *a.total = all;
  }
  __syncthreads();
  int* const went = a.first ? a.place : a.went;
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const unsigned i = tile0 + w * (64 * IPT) + r * 64 + lane, key = (unsigned)(pair[r] >> 32);
    int to = -1;
    if (key != kGroupNone) {
      const unsigned d = (key >> a.shift) & mask, p = whist[w][d] + rank[r];
      tile[p] = pair[r];
      to = (int)(base[d] + p);
    }
    if (i < N) went[i] = to;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < IPT; ++r) {
    const unsigned p = r * kGroupThreads + tid;
    if (p < in_tile) {
      const unsigned long long v = tile[p];
      const unsigned key = (unsigned)(v >> 32), to = base[(key >> a.shift) & mask] + p;
      if (a.last) {
        a.order[to] = (int)(unsigned)v;
        if (a.key_out) a.key_out[to] = key;
      } else {
        a.pair_out[to] = v;
      }
    }
    if (a.last && tile0 + p >= all && tile0 + p < a.in.N) a.order[tile0 + p] = -1;
  }
}

// The end of a sort of several passes, two jobs side by side: workgroups below `follow` follow the passes behind the first one, place[i] =
// went2[went1[place[i]]], four entries per thread; the others find offsets[e] = entries whose key is below e in the sorted keys.
// start: first slot of every bin of the last pass (keys >> shift), or null.  A bin of at most 2048 lists and four entries to a list is read
// once: where a key differs from the one before it a list starts, and a list that does not is empty and starts where the next one does.
// Else a binary search per list.  Reading / searching, the whole sort: 2^20 entries by 2^20 lists 60.7 / 67.0 us, 2^18 35.6 / 41.1; with
// sixteen entries to a list 2^20 by 65536 54.0 / 51.3.
// first of keys[lo, hi) that is not below e
__device__ __forceinline__ unsigned group_lower(const unsigned* keys, unsigned lo, unsigned hi, unsigned e) {
  while (lo < hi) {
    const unsigned mid = lo + (hi - lo) / 2;
    if (keys[mid] < e) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(256) group_end_kernel(unsigned follow, int* place, const int* went1, const int* went2, unsigned N,
                                                        const unsigned* keys, const unsigned* total, const unsigned* start, int shift,
                                                        int* offsets, unsigned E) {
  if (blockIdx.x < follow) {
    const unsigned i0 = blockIdx.x * 1024u + threadIdx.x;
    int p[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = i0 + r * 256 < N ? place[i0 + r * 256] : -1;
#pragma unroll
    for (int r = 0; r < 4; ++r) p[r] = p[r] >= 0 ? went1[p[r]] : -1;
    if (went2) {
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = p[r] >= 0 ? went2[p[r]] : -1;
    }
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if (i0 + r * 256 < N) place[i0 + r * 256] = p[r];
    return;
  }
  const unsigned all = *total, block = blockIdx.x - follow, blocks = gridDim.x - follow;
  if (block == 0 && threadIdx.x == 0) offsets[E] = (int)all;
  if (start && shift <= kGroupMaxBits) {   // a workgroup per bin
    __shared__ unsigned first[kGroupMaxBins], tail[4];
    const unsigned lists = 1u << shift, e0 = block << shift, lo = start[block], hi = start[block + 1];
    if (hi - lo <= 4 * lists) {
      for (unsigned j = threadIdx.x; j < kGroupMaxBins; j += 256) first[j] = hi;
      __syncthreads();
      for (unsigned i = lo + threadIdx.x; i < hi; i += 256) {
        const unsigned k = keys[i];
        if (i == lo || keys[i - 1] != k) first[k - e0] = i;
      }
      __syncthreads();
      // smallest of all behind: eight neighbouring lists per thread, then the threads behind it
      unsigned v[kGroupMaxBins / 256], m = hi;
#pragma unroll
      for (int j = kGroupMaxBins / 256 - 1; j >= 0; --j) v[j] = m = min(m, first[threadIdx.x * (kGroupMaxBins / 256) + j]);
      const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
      for (int d = 1; d < 64; d <<= 1) {
        const unsigned o = __shfl_down(m, d, 64);
        if (lane + d < 64) m = min(m, o);
      }
      if (lane == 0) tail[w] = m;
      unsigned behind = __shfl_down(m, 1, 64);
      __syncthreads();
      if (lane == 63) behind = hi;
      for (int o = w + 1; o < 4; ++o) behind = min(behind, tail[o]);
#pragma unroll
      for (int j = 0; j < kGroupMaxBins / 256; ++j) {
        const unsigned at = threadIdx.x * (kGroupMaxBins / 256) + j;
        first[at] = min(v[j], behind);
      }
      __syncthreads();
      for (unsigned j = threadIdx.x; j < lists && e0 + j < E; j += 256) offsets[e0 + j] = (int)first[j];
      return;
    }
    for (unsigned j = threadIdx.x; j < lists && e0 + j < E; j += 256) offsets[e0 + j] = (int)group_lower(keys, lo, hi, e0 + j);
    return;
  }
  for (unsigned long e = block * 256ul + threadIdx.x; e < E; e += blocks * 256ul)
    offsets[e] = (int)group_lower(keys, start ? start[e >> shift] : 0, start ? start[(e >> shift) + 1] : all, (unsigned)e);
}

// Up to one tile of entries: every pass in one workgroup, keys and entries in LDS between the passes.
__global__ void __launch_bounds__(kGroupThreads) group_small_kernel(GroupPass a, int passes) {
  __shared__ unsigned skey[kGroupTile];
  __shared__ unsigned short sidx[kGroupTile];
  __shared__ unsigned short whist[kGroupWaves][kGroupMaxBins];
  __shared__ unsigned base[kGroupMaxBins];
  __shared__ unsigned tmp[kGroupWaves];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int bins = 1 << a.bits;
  const unsigned mask = bins - 1;
  const int rounds = (int)((a.in.N + kGroupThreads - 1) / kGroupThreads);   // entries per thread, the same for every wave
  unsigned n = a.in.N;
  unsigned key[kGroupIpt], rank[kGroupIpt];
  int idx[kGroupIpt];
  bool any_bad = false;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * a.bits;
    for (int b = tid; b < bins; b += kGroupThreads)
      for (int v = 0; v < kGroupWaves; ++v) whist[v][b] = 0;
#pragma unroll
    for (int r = 0; r < kGroupIpt; ++r) {
      const unsigned i = (w * rounds + r) * 64 + lane;
      key[r] = kGroupNone;
      idx[r] = (int)i;
      if (r < rounds && i < n) {
        if (pass == 0) {
          bool bad;
          key[r] = group_key(a.in, i, bad);
          any_bad |= bad;
          if (key[r] == kGroupNone) a.place[i] = -1;
        } else {
          key[r] = skey[i];
          idx[r] = sidx[i];
        }
      }
    }
    __syncthreads();
    auto key_of = [&](int r) { return key[r]; };
    if (a.bits <= 8) group_rank<8>(whist[w], key_of, shift, mask, rank, rounds);
    else group_rank<kGroupMaxBits>(whist[w], key_of, shift, mask, rank, rounds);
    __syncthreads();
    const int bpt = (bins + kGroupThreads - 1) / kGroupThreads;
    unsigned mine[kGroupMaxBins / kGroupThreads], s = 0;
#pragma unroll
    for (int j = 0; j < kGroupMaxBins / kGroupThreads; ++j) {
      const int b = tid * bpt + j;
      mine[j] = 0;
      if (j < bpt && b < bins) {
        unsigned run = 0;
        for (int v = 0; v < kGroupWaves; ++v) {
          const unsigned c = whist[v][b];
          whist[v][b] = (unsigned short)run;
          run += c;
        }
        mine[j] = run;
      }
      s += mine[j];
    }
    unsigned all;
    unsigned start = group_block_scan(s, tmp, &all);
#pragma unroll
    for (int j = 0; j < kGroupMaxBins / kGroupThreads; ++j) {
      const int b = tid * bpt + j;
      if (j < bpt && b < bins) {
        base[b] = start;
        start += mine[j];
      }
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kGroupIpt; ++r) {
      if (r < rounds && key[r] != kGroupNone) {
        const unsigned d = (key[r] >> shift) & mask;
        const unsigned dst = base[d] + whist[w][d] + rank[r];
        skey[dst] = key[r];
        sidx[dst] = (unsigned short)idx[r];
      }
    }
    n = all;
    __syncthreads();
  }
  if (any_bad && a.bad) *a.bad = 1;
  for (unsigned p = tid; p < a.in.N; p += kGroupThreads) {
    if (p < n) {
      const int i = sidx[p];
      a.order[p] = i;
      a.place[i] = (int)p;
      if (a.key_out) a.key_out[p] = skey[p];
    } else {
      a.order[p] = -1;
    }
  }
  if (tid == 0 && a.total) *a.total = n;
  if (a.offsets)
    for (unsigned e = tid; e <= a.in.E; e += kGroupThreads) {
      unsigned lo = 0, hi = n;
      while (lo < hi) {
        const unsigned mid = (lo + hi) / 2;
        if (skey[mid] < e) lo = mid + 1;
        else hi = mid;
      }
      a.offsets[e] = (int)lo;
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Rows.  All of these are bound by HBM: a row is read or written once, in units of 16 bytes whatever its alignment (the hardware takes
// 16-byte accesses at any element); the last unit ends with the row and overlaps the one before it.  Rows shorter than that go element by
// element (E = 1).  `lanes` (a power of two up to 64) lanes share a row and step through its units, so no index is divided.
// ---------------------------------------------------------------------------------------------------------------------
struct GroupRows {
  const int* place;    // (n, k)
  const int* end;      // = offsets + E: slots in use
  long n, N;           // rows, entries = n k
  int k;
  int D, units;        // elements and units per row
  int lanes_log2;
};

// slot of an entry, -1 without one (and for what cannot be a slot: nothing is read or written out of bounds whatever `place` holds)
__device__ __forceinline__ int group_place(const GroupRows& g, long r, int j) {
  const int p = g.place[r * g.k + j];
  return (unsigned)p < (unsigned)g.N ? p : -1;
}

template <typename T, int E>
struct GroupUnit {
  struct alignas(sizeof(T)) Raw { T v[E]; };
  T v[E];
  __device__ __forceinline__ void load(const T* at) {
    const Raw r = *reinterpret_cast<const Raw*>(at);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = r.v[e];
  }
  __device__ __forceinline__ void store(T* at) const {
    Raw r;
#pragma unroll
    for (int e = 0; e < E; ++e) r.v[e] = v[e];
    *reinterpret_cast<Raw*>(at) = r;
  }
};

// T: an unsigned type, the widest (up to 8 bytes) that rows, strides and bases are multiples of
template <typename T, int E>
__global__ void __launch_bounds__(256) group_gather_kernel(GroupRows g, const T* x, long x_stride, T* out) {
  const int lanes = 1 << g.lanes_log2;
  const int u0 = threadIdx.x & (lanes - 1);
  const long per = 256 >> g.lanes_log2;
  const long first = (long)blockIdx.x * per + (threadIdx.x >> g.lanes_log2), step = (long)gridDim.x * per;
  GroupUnit<T, E> v;
  for (long r = first; r < g.n; r += step) {
    const int* pl = g.place + r * g.k;
    for (int u = u0; u < g.units; u += lanes) {
      const int at = min(u * E, g.D - E);
      v.load(x + r * x_stride + at);
      for (int j = 0; j < g.k; ++j) {
        const int p = pl[j];
        if ((unsigned)p < (unsigned)g.N) v.store(out + (long)p * g.D + at);
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e) v.v[e] = T{};
  for (long s = max(*g.end, 0) + first; s < g.N; s += step)
    for (int u = u0; u < g.units; u += lanes) v.store(out + s * g.D + min(u * E, g.D - E));
}

// Rows of one element (at most 8 bytes: a row of byte codes), a slot per thread: neighbouring stores and scattered reads, which the cache
// serves, where the kernel above has it the other way round.  10^6 rows of 8 bytes 13.0 / 14.8 us (14.2 / 13.8 with nothing in the cache),
// 262144 x 4 of them 6.7 / 14.4; of 16 bytes 18.2 / 15.7 (k = 1).
template <typename T>
__global__ void __launch_bounds__(256) group_pull_kernel(GroupRows g, const int* order, const T* x, long x_stride, T* out) {
  const long end = min((long)max(*g.end, 0), g.N);
  for (long s = blockIdx.x * 256l + threadIdx.x; s < g.N; s += gridDim.x * 256l) {
    const unsigned e = s < end ? (unsigned)order[s] : ~0u;
    out[s] = e < (unsigned)g.N ? x[(long)(g.k == 1 ? e : e / (unsigned)g.k) * x_stride] : T{};
  }
}

template <typename T> struct GroupNum;
template <> struct GroupNum<float> {
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct GroupNum<_Float16> {
  static __device__ __forceinline__ float get(_Float16 v) { return (float)v; }
  static __device__ __forceinline__ _Float16 put(float v) { return (_Float16)v; }
};
template <> struct GroupNum<__bf16> {
  static __device__ __forceinline__ float get(__bf16 v) { return (float)v; }
  static __device__ __forceinline__ __bf16 put(float v) { return (__bf16)v; }
};

// weight of entry i in 32 bits (w_dtype: QINCO_T_*; no weights: 1)
__device__ __forceinline__ float group_weight(const void* w, int w_dtype, long i) {
  if (!w) return 1.f;
  if (w_dtype == 0) return reinterpret_cast<const float*>(w)[i];
  if (w_dtype == 1) return (float)reinterpret_cast<const _Float16*>(w)[i];
  return (float)reinterpret_cast<const __bf16*>(w)[i];
}

// out[r] = sum_j w[r, j] y[place[r, j]]: sums in 32 bits in the order of j, rounded once.  The gradient of the gather is this with
// weights of one.  J entries of a row are loaded before the first one is used.
template <typename T, int E, int J>
__global__ void __launch_bounds__(256) group_combine_kernel(GroupRows g, const T* y, long y_stride, const void* wt, int w_dtype, T* out) {
  const int lanes = 1 << g.lanes_log2;
  const int u0 = threadIdx.x & (lanes - 1);
  const long per = 256 >> g.lanes_log2;
  const long first = (long)blockIdx.x * per + (threadIdx.x >> g.lanes_log2), step = (long)gridDim.x * per;
  for (long r = first; r < g.n; r += step) {
    for (int u = u0; u < g.units; u += lanes) {
      const int at = min(u * E, g.D - E);
      float acc[E];
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] = 0.f;
      for (int j0 = 0; j0 < g.k; j0 += J) {
        int p[J];
        float w[J];
        GroupUnit<T, E> v[J];
#pragma unroll
        for (int j = 0; j < J; ++j) p[j] = j0 + j < g.k ? group_place(g, r, j0 + j) : -1;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (p[j] >= 0) {
            w[j] = group_weight(wt, w_dtype, r * g.k + j0 + j);
            v[j].load(y + (long)p[j] * y_stride + at);
          }
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
          if (p[j] >= 0) {
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = fmaf(w[j], GroupNum<T>::get(v[j].v[e]), acc[e]);
          }
        }
      }
      GroupUnit<T, E> o;
#pragma unroll
      for (int e = 0; e < E; ++e) o.v[e] = GroupNum<T>::put(acc[e]);
      o.store(out + r * g.D + at);
    }
  }
}

// sum over the 2^lanes_log2 neighbouring lanes of a row: inside 16 lanes by DPP (swap neighbours, swap pairs, mirror halves, mirror)
template <int CTRL>
__device__ __forceinline__ float group_dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false));
}
__device__ __forceinline__ float group_lanes_sum(float v, int lanes_log2) {
  if (lanes_log2 > 0) v += group_dpp<0xB1>(v);
  if (lanes_log2 > 1) v += group_dpp<0x4E>(v);
  if (lanes_log2 > 2) v += group_dpp<0x141>(v);
  if (lanes_log2 > 3) v += group_dpp<0x140>(v);
  if (lanes_log2 > 4) v += __shfl_xor(v, 16, 64);
  if (lanes_log2 > 5) v += __shfl_xor(v, 32, 64);
  return v;
}

// dy[place[r, j]] = w[r, j] dout[r], dw[r, j] = <dout[r], y[place[r, j]]> in one pass over y and dout; rows of dy no entry owns: zeros.
// Two entries at a time (1 / 2 / 4 / 8: 65536 rows of 8 x 128 bf16 68 / 76 / 72 / 77 us, fp32 155 / 127 / 128 / 129, 2 x 768 bf16
// 104 / 113 / 131 / 191, 4096 rows of 4 x 384 fp32 13.3 / 12.3 / 12.3 / 13.6): more take registers and with them waves.
template <typename T, int E, typename W>
__global__ void __launch_bounds__(256) group_combine_grad_kernel(GroupRows g, const T* dout, long dout_stride, const T* y, long y_stride,
                                                                 const W* wt, T* dy, W* dw) {
  constexpr int J = 2;
  const int lanes = 1 << g.lanes_log2;
  const int u0 = threadIdx.x & (lanes - 1);
  const long per = 256 >> g.lanes_log2;
  const long first = (long)blockIdx.x * per + (threadIdx.x >> g.lanes_log2), step = (long)gridDim.x * per;
  // (the loop over rows is taken by whole waves: the sums over a row's lanes want all of them active)
  const long rounds = (g.n + step - 1) / step;
  for (long i = 0; i < rounds; ++i) {
    const long r = first + i * step;
    for (int j0 = 0; j0 < g.k; j0 += J) {
      int p[J];
      float w[J], dot[J];
#pragma unroll
      for (int j = 0; j < J; ++j) p[j] = r < g.n && j0 + j < g.k ? group_place(g, r, j0 + j) : -1;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        w[j] = dy && p[j] >= 0 ? GroupNum<W>::get(wt[r * g.k + j0 + j]) : 0.f;
        dot[j] = 0.f;
      }
      if (r < g.n) {
        for (int u = u0; u < g.units; u += lanes) {
          const int at = min(u * E, g.D - E);
          GroupUnit<T, E> d, v[J];
          d.load(dout + r * dout_stride + at);
          if (dw) {
#pragma unroll
            for (int j = 0; j < J; ++j)
              if (p[j] >= 0) v[j].load(y + (long)p[j] * y_stride + at);
          }
          if (dy) {
#pragma unroll
            for (int j = 0; j < J; ++j) {
              if (p[j] >= 0) {
                GroupUnit<T, E> o;
#pragma unroll
                for (int e = 0; e < E; ++e) o.v[e] = GroupNum<T>::put(w[j] * GroupNum<T>::get(d.v[e]));
                o.store(dy + (long)p[j] * g.D + at);
              }
            }
          }
          if (dw) {
            if (at < u * E) {   // the last unit's overlap counts once: zeros on both sides (0 inf would be NaN)
#pragma unroll
              for (int e = 0; e < E; ++e) {
                if (at + e < u * E) {
                  d.v[e] = T{};
#pragma unroll
                  for (int j = 0; j < J; ++j) v[j].v[e] = T{};
                }
              }
            }
            float x[E];
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = GroupNum<T>::get(d.v[e]);
#pragma unroll
            for (int j = 0; j < J; ++j) {
              if (p[j] >= 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) dot[j] = fmaf(x[e], GroupNum<T>::get(v[j].v[e]), dot[j]);
              }
            }
          }
        }
      }
      if (dw) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float s = group_lanes_sum(dot[j], g.lanes_log2);
          if (u0 == 0 && r < g.n && j0 + j < g.k) dw[r * g.k + j0 + j] = GroupNum<W>::put(s);
        }
      }
    }
  }
  if (!dy) return;
  GroupUnit<T, E> zero;
#pragma unroll
  for (int e = 0; e < E; ++e) zero.v[e] = T{};
  for (long s = max(*g.end, 0) + first; s < g.N; s += step)
    for (int u = u0; u < g.units; u += lanes) zero.store(dy + s * g.D + min(u * E, g.D - E));
}

}  // namespace qinco
