// C ABI of the operators between a model that answers in codes and the codec (include/qinco_hip.h): codes drawn from logits
// (sample_kernel.hpp) and rows grouped by inverted list (group_kernel.hpp).  None of them keeps state: outputs and workspace are the
// caller's, every argument is checked on the host before anything is launched, and nothing is synchronised.
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "abi_util.hpp"
#include "group_kernel.hpp"
#include "sample_kernel.hpp"

using namespace qinco;
#define fail qinco::abi_fail

static constexpr int64_t kMaxLists = (int64_t)1 << 24;

static int bits_of(uint64_t v) {   // bits that hold 0 .. v - 1
  int b = 0;
  while (b < 63 && ((uint64_t)1 << b) < v) ++b;
  return b;
}

static bool known(int dtype) { return dtype == QINCO_T_F32 || dtype == QINCO_T_F16 || dtype == QINCO_T_BF16; }

// a workspace holds whole numbers of 64 bits and takes atomics: at an odd address these would fault
static bool aligned(const void* ws) { return reinterpret_cast<uintptr_t>(ws) % 16 == 0; }

// ---------------------------------------------------------------------------------------------
// sampling
// ---------------------------------------------------------------------------------------------
static constexpr long kCUs = 256;
static constexpr int kSampleBlockThreads = 1024, kSampleBlockCodes = 20;   // the largest workgroup per row, and codes per thread
// V above which a row is split over workgroups
static constexpr int64_t kSampleLongV = kSampleBlockThreads * kSampleBlockCodes;

namespace {
struct SamplePlan {
  int64_t rows, chunks;                                                          // rows of a batch
  int64_t most;                                                                  // members that a row's list holds
  int64_t best, least, sum, floor, mass, count, row_mass, row_count, state, chunk_mass, m_z, m_where, bytes;   // byte offsets
};
}  // namespace

// Rows go through in batches whose workspace stays within 128 MiB (what one kernel writes the next finds in the 256 MiB cache), one row at
// least.  A row's list holds an eighth of it: bins that the cuts fall into hold more only where that many logits are next to each other.
static SamplePlan sample_plan(int64_t n, int64_t V) {
  SamplePlan p{};
  if (V <= kSampleLongV) return p;
  p.chunks = (V + kSampleChunk - 1) / kSampleChunk;
  p.most = V / 8 > 2 * kSampleMembers ? V / 8 : 2 * kSampleMembers;
  p.rows = ((int64_t)128 << 20) / (p.chunks * kSampleBins * 12 + kSampleBins * 12 + p.most * 8);
  if (p.rows < 1) p.rows = 1;
  if (p.rows > n) p.rows = n;
  int64_t at = 0;
  auto take = [&](int64_t& o, int64_t bytes) {
    o = at;
    at += (bytes + 255) / 256 * 256;
  };
  const int64_t R = p.rows, RC = R * p.chunks;
  take(p.best, RC * 8);
  take(p.least, RC * 4);
  take(p.sum, RC * 4);
  take(p.floor, RC * 4);
  take(p.mass, RC * kSampleBins * 8);
  take(p.count, RC * kSampleBins * 4);
  take(p.row_mass, R * kSampleBins * 8);
  take(p.row_count, R * kSampleBins * 4);
  take(p.state, R * (int64_t)sizeof(SampleState));
  take(p.chunk_mass, RC * 8);
  take(p.m_z, R * p.most * 4);
  take(p.m_where, R * p.most * 4);
  p.bytes = at;
  return p;
}

extern "C" int64_t qinco_sample_workspace(int64_t n, int64_t V) {
  if (n < 0 || V < 1 || V > kMaxLists) return 0;
  return sample_plan(n, V).bytes;
}

template <typename T>
static int launch_sample_long(const SampleArgs& a, const SamplePlan& p, char* ws, hipStream_t st) {
  SampleLong l{};
  l.chunks = (int)p.chunks;
  l.best = reinterpret_cast<unsigned long long*>(ws + p.best);
  l.least = reinterpret_cast<unsigned*>(ws + p.least);
  l.sum = reinterpret_cast<float*>(ws + p.sum);
  l.floor = reinterpret_cast<int*>(ws + p.floor);
  l.mass = reinterpret_cast<unsigned long long*>(ws + p.mass);
  l.count = reinterpret_cast<unsigned*>(ws + p.count);
  l.row_mass = reinterpret_cast<unsigned long long*>(ws + p.row_mass);
  l.row_count = reinterpret_cast<unsigned*>(ws + p.row_count);
  l.state = reinterpret_cast<SampleState*>(ws + p.state);
  l.chunk_mass = reinterpret_cast<unsigned long long*>(ws + p.chunk_mass);
  l.m_z = reinterpret_cast<float*>(ws + p.m_z);
  l.m_where = reinterpret_cast<unsigned*>(ws + p.m_where);
  l.most = (int)p.most;
  l.uncut = !a.k_rows && !a.p_rows && !a.m_rows && (a.k <= 0 || a.k >= a.V) && a.p >= 1.0 && !(a.m > 0.0);
  for (long r0 = 0; r0 < a.n; r0 += p.rows) {
    const long rows = a.n - r0 < p.rows ? a.n - r0 : (long)p.rows;
    l.row0 = r0;
    const dim3 grid((unsigned)(rows * p.chunks)), block(kSampleChunkThreads);
    hipLaunchKernelGGL(sample_range_kernel<T>, grid, block, 0, st, a, l);
    HIP_TRY(hipGetLastError());
    if (l.uncut) {
      hipLaunchKernelGGL(sample_mass_kernel<T>, grid, block, 0, st, a, l);
      HIP_TRY(hipGetLastError());
    } else {
      hipLaunchKernelGGL(sample_bins_kernel<T>, grid, block, 0, st, a, l);
      HIP_TRY(hipGetLastError());
      if (p.chunks > kSampleFewChunks) {
        hipLaunchKernelGGL(sample_sum_bins_kernel, dim3((unsigned)(rows * (kSampleBins / 64))), dim3(1024), 0, st, l);
        HIP_TRY(hipGetLastError());
      }
      hipLaunchKernelGGL(sample_cuts_kernel, dim3((unsigned)rows), dim3(1024), 0, st, a, l);
      HIP_TRY(hipGetLastError());
      hipLaunchKernelGGL(sample_members_kernel<T>, grid, block, 0, st, a, l);
      HIP_TRY(hipGetLastError());
    }
    hipLaunchKernelGGL(sample_finish_kernel<T>, dim3((unsigned)rows), block, 0, st, a, l);
    HIP_TRY(hipGetLastError());
  }
  return QINCO_OK;
}

// f(workgroups, first row): launches of `rows` rows per workgroup of `threads`, each of fewer than 2^32 threads.  (A loop over rows inside the
// kernels would have the compiler take what all rows share out of it, into registers that the rows' own values need.)
template <typename F>
static void sample_launches(int64_t n, int rows, int threads, F f) {
  const int64_t most = ((int64_t)1 << 31) / threads * rows;
  for (int64_t r0 = 0; r0 < n; r0 += most) f(dim3((unsigned)(((n - r0 < most ? n - r0 : most) + rows - 1) / rows)), (long)r0);
}

template <typename T, int R>
static void launch_sample_wave(const SampleArgs& a, hipStream_t st) {
  sample_launches(a.n, kSampleRowWaves, 64 * kSampleRowWaves, [&](dim3 grid, long r0) {
    hipLaunchKernelGGL((sample_wave_kernel<T, R>), grid, dim3(64 * kSampleRowWaves), 0, st, a, r0);
  });
}

template <typename T, int G, int R>
static void launch_sample_group(const SampleArgs& a, hipStream_t st) {
  sample_launches(a.n, kSampleGroupThreads / G, kSampleGroupThreads, [&](dim3 grid, long r0) {
    hipLaunchKernelGGL((sample_group_kernel<T, G, R>), grid, dim3(kSampleGroupThreads), 0, st, a, r0);
  });
}

template <typename T, int NT, int R>
static void launch_sample_block(const SampleArgs& a, hipStream_t st) {
  sample_launches(a.n, 1, NT, [&](dim3 grid, long r0) { hipLaunchKernelGGL((sample_block_kernel<T, NT, R>), grid, dim3(NT), 0, st, a, r0); });
}

// By the length of a row, and where the rows alone do not fill the card with more lanes to each (a row's code depends on neither).  Both sides of
// each border measured, all three cuts on, fp32.  65536 rows of 64 24 us with 4 codes per lane, 35 with 8; of 128 38 us with 16 lanes, 68 with
// 32; of 256 70 us with 32, 81 with 64.  With a wave each or fewer lanes, one row of 128 or 256 4.8 and 6.5 us, 2048 rows of 256 6.9 and 7.8,
// 4096 9.0 and 8.7; 2048 of 128 6.3 and 7.8, 8192 13.0 and 8.6.  16384 of 512 38 us with a wave each, 82 with four; of 1000 97 us with 4 codes
// per thread, 113 with 8; 8000 of 2000 75 us with 8, 89 with 20; of 4099 136 us with 256 threads, 182 with 512; of 10240 289 us with 512 threads,
// 474 with 1024; one row of 20480 21 us with a workgroup, 43 split over several, 1000 of them 97 and 190.  Few rows, 512 and 256 threads: of 2000
// one 7.8 and 9.1 us, 256 8.5 and 9.9, 500 10.5 and 11.0, 700 12.6 and 12.1, 1000 16.6 and 13.6; of 4099 one 10.8 and 13.9, 256 11.6 and 14.8, 500
// 14.6 and 16.8, 700 22.0 and 19.3, 1000 26 and 22; 1024 and 512 threads, of 10240 one 14.9 and 15.6, 256 16.1 and 17.1, 300 29 and 22.  (So up to
// 6144 codes the border of one row per CU comes early: at two the larger workgroups are still 5 to 15 % ahead.)
template <typename T>
static int launch_sample(const SampleArgs& a, const SamplePlan& p, char* ws, hipStream_t st) {
  if (a.V > kSampleLongV) return launch_sample_long<T>(a, p, ws, st);
  if (a.V <= 64) launch_sample_group<T, 16, 4>(a, st);
  else if (a.n <= 8 * kCUs && a.V <= 256) launch_sample_wave<T, 4>(a, st);   // (two waves per SIMD)
  else if (a.V <= 128) launch_sample_group<T, 16, 8>(a, st);
  else if (a.V <= 256) launch_sample_group<T, 32, 8>(a, st);
  else if (a.V <= 512) launch_sample_wave<T, 8>(a, st);
  else if (a.V <= 256 * 4) launch_sample_block<T, 256, 4>(a, st);
  else if (a.n <= kCUs && a.V <= 512 * 4) launch_sample_block<T, 512, 4>(a, st);
  else if (a.n <= kCUs && a.V <= 512 * 12) launch_sample_block<T, 512, 12>(a, st);
  else if (a.V <= 256 * 8) launch_sample_block<T, 256, 8>(a, st);
  else if (a.V <= 256 * 20) launch_sample_block<T, 256, 20>(a, st);
  else if (a.n > kCUs && a.V <= 512 * 20) launch_sample_block<T, 512, 20>(a, st);
  else launch_sample_block<T, kSampleBlockThreads, kSampleBlockCodes>(a, st);
  HIP_TRY(hipGetLastError());
  return QINCO_OK;
}

extern "C" int qinco_sample_codes(const void* logits, int dtype, int64_t row_stride, int64_t n, int64_t V, const void* u, int u_is_f64,
                                  const qinco_sample_params* params, void* codes_out, int code_dtype, float* logp_out, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  if (!params || params->struct_bytes != (int32_t)sizeof(qinco_sample_params))
    return fail(QINCO_ERR_INVALID, "qinco_sample_codes: params missing, or struct_bytes is not sizeof(qinco_sample_params)");
  if (!known(dtype)) return fail(QINCO_ERR_INVALID, "qinco_sample_codes: unknown element type %d", dtype);
  if (code_dtype != QINCO_CODE_I64 && code_dtype != QINCO_CODE_I32)
    return fail(QINCO_ERR_INVALID, "qinco_sample_codes: codes are int64 or int32 (a row with nothing to draw answers -1)");
  if (V < 1 || V > kMaxLists) return fail(QINCO_ERR_INVALID, "qinco_sample_codes: need 1 <= V <= 2^24 (V=%lld)", (long long)V);
  if (n < 0 || n > INT32_MAX) return fail(QINCO_ERR_INVALID, "qinco_sample_codes: need 0 <= n < 2^31 (n=%lld)", (long long)n);
  if (row_stride < 0) return fail(QINCO_ERR_INVALID, "qinco_sample_codes: negative row stride");
  if (n == 0) return QINCO_OK;
  if (!logits || !u || !codes_out) return fail(QINCO_ERR_INVALID, "qinco_sample_codes: null buffer");
  const SamplePlan p = sample_plan(n, V);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return fail(QINCO_ERR_INVALID, "qinco_sample_codes: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.bytes);
  if (p.bytes > 0 && !aligned(workspace)) return fail(QINCO_ERR_INVALID, "qinco_sample_codes: workspace not aligned to 16 bytes");
  const int lv = bits_of((uint64_t)V);
  SampleArgs a{logits, (long)row_stride, (long)n, (int)V, u, u_is_f64 != 0, params->temperature_rows, params->temperature, params->top_k_rows,
               params->top_k, params->top_p_rows, params->top_p, params->min_p_rows, params->min_p, codes_out,
               code_dtype == QINCO_CODE_I64, logp_out, lv > 0 ? lv - 1 : 0};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  char* ws = reinterpret_cast<char*>(workspace);
  if (dtype == QINCO_T_F32) return launch_sample<float>(a, p, ws, st);
  if (dtype == QINCO_T_F16) return launch_sample<_Float16>(a, p, ws, st);
  return launch_sample<__bf16>(a, p, ws, st);
}

// ---------------------------------------------------------------------------------------------
// grouping
// ---------------------------------------------------------------------------------------------
namespace {
struct GroupPlan {
  int bits, passes;                                       // bits of one digit (the same for every pass)
  int ipt;
  int64_t tiles;
  int64_t totals, start, counts, pairs, keys, went, words;   // workspace in 32-bit words (the total of entries is its first)
};
}  // namespace

// Counts (tiles times bins) up to which every workgroup of the scatter sums them itself, a launch less per pass (summed there / by a kernel of
// their own: 16384 entries by 1024 lists, 16 tiles of 1024 bins, 10.2 / 11.5 us, 32768 12.1 / 11.6; by 65536 lists, two passes of 256 bins, 32
// tiles 20.8 / 23.8, 64 24.1 / 24.8, 96 27.7 / 25.5; 8192 by 2048 12.6 / 12.9, 16384 16.2 / 13.0)
static constexpr int64_t kGroupFewCounts = 1 << 14;

// Entries per thread.  A tile has a cost of its own (tables of its digits), few tiles leave the chip empty.  Measured with 2 / 4 / 8 per
// thread, a sort by 1024 lists: 2^17 entries 12.6 / 14.4 / 18.9 us, 2^18 14.4 / 15.4 / 19.5, 2^19 23.3 / 17.9 / 20.7, 2^20 43.4 / 28.4 / 24.5,
// 2^22 151 / 104 / 67.
static GroupPlan group_plan(int64_t N, int64_t E) {
  GroupPlan p{};
  const int all = bits_of((uint64_t)E);
  p.passes = all <= kGroupMaxBits ? 1 : (all + kGroupMaxBits - 1) / kGroupMaxBits;
  p.bits = (all + p.passes - 1) / p.passes;
  p.ipt = N <= (1 << 18) ? 2 : N <= (1 << 19) ? 4 : 8;
  p.tiles = (N + kGroupThreads * p.ipt - 1) / (kGroupThreads * p.ipt);
  const int64_t bins = (int64_t)1 << p.bits;
  const bool small = N <= kGroupTile;
  int64_t at = 16;
  auto take = [&](int64_t& o, int64_t words) {
    o = at;
    at += (words + 15) / 16 * 16;
  };
  take(p.totals, small ? 0 : bins);
  take(p.start, small ? 0 : bins + 1);
  take(p.counts, small ? 0 : p.tiles * bins);
  take(p.pairs, small || p.passes == 1 ? 0 : 2 * N * (p.passes == 2 ? 1 : 2));
  take(p.keys, (small ? E > kGroupSmallOffsets : p.passes > 1) ? N : 0);
  take(p.went, small ? 0 : N * (p.passes - 1));
  p.words = at;
  return p;
}

extern "C" int64_t qinco_group_workspace(int64_t entries, int64_t n_lists) {
  if (entries < 0 || entries > INT32_MAX || n_lists < 1 || n_lists > kMaxLists) return 0;
  return group_plan(entries, n_lists).words * 4;
}

template <typename F>
static void with_ipt(int ipt, F f) {
  if (ipt == 2) f(std::integral_constant<int, 2>{});
  else if (ipt == 4) f(std::integral_constant<int, 4>{});
  else f(std::integral_constant<int, 8>{});
}

// N entries to follow (0: none), E + 1 offsets to find
static int launch_end(int* place, const int* went1, const int* went2, int64_t N, const unsigned* keys, const unsigned* total,
                      const unsigned* start, int shift, int* offsets, unsigned E, hipStream_t st) {
  const unsigned follow = (unsigned)((N + 1023) / 1024);
  long g = ((long)E + 256) / 256;
  if (g > 4096) g = 4096;
  if (start && shift <= kGroupMaxBits) g = ((long)E + (1 << shift) - 1) >> shift;   // a workgroup per bin
  hipLaunchKernelGGL(group_end_kernel, dim3(follow + (unsigned)g), dim3(256), 0, st, follow, place, went1, went2, (unsigned)N, keys, total,
                     start, shift, offsets, E);
  HIP_TRY(hipGetLastError());
  return QINCO_OK;
}

extern "C" int qinco_group_rows(const void* lists, int code_dtype, int64_t row_stride, int64_t n, int32_t k, int64_t n_lists, int32_t* order,
                                int32_t* place, int32_t* offsets, int32_t* bad, void* workspace, int64_t workspace_bytes, void* stream) {
  if (code_dtype != QINCO_CODE_I64 && code_dtype != QINCO_CODE_I32 && code_dtype != QINCO_CODE_U8)
    return fail(QINCO_ERR_INVALID, "qinco_group_rows: unknown code type %d", code_dtype);
  if (n_lists < 1 || n_lists > kMaxLists)
    return fail(QINCO_ERR_INVALID, "qinco_group_rows: need 1 <= n_lists <= 2^24 (n_lists=%lld)", (long long)n_lists);
  if (n < 0 || k < 1 || n > INT32_MAX / k) return fail(QINCO_ERR_INVALID, "qinco_group_rows: need n >= 0, k >= 1, n k < 2^31");
  if (row_stride < 0) return fail(QINCO_ERR_INVALID, "qinco_group_rows: negative row stride");
  const int64_t N = n * k;
  if (!offsets || (N > 0 && (!lists || !order || !place))) return fail(QINCO_ERR_INVALID, "qinco_group_rows: null buffer");
  const GroupPlan p = group_plan(N, n_lists);
  if (!workspace || workspace_bytes < p.words * 4)
    return fail(QINCO_ERR_INVALID, "qinco_group_rows: workspace of %lld bytes, %lld needed", (long long)workspace_bytes, (long long)p.words * 4);
  if (!aligned(workspace)) return fail(QINCO_ERR_INVALID, "qinco_group_rows: workspace not aligned to 16 bytes");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  unsigned* ws = reinterpret_cast<unsigned*>(workspace);
  const unsigned E = (unsigned)n_lists;
  GroupPass a{};
  a.in = GroupKeys{lists, code_dtype, (long)row_stride, (unsigned)k, (unsigned)N, E};
  a.place = place;
  a.order = order;
  a.total = ws;
  a.totals = ws + p.totals;
  a.counts = ws + p.counts;
  a.bad = bad;
  a.bits = p.bits;
  a.first = a.last = 1;
  a.tiles = p.tiles << p.bits <= kGroupFewCounts ? (int)p.tiles : 0;
  if (N <= kGroupTile) {
    const bool search = E > (unsigned)kGroupSmallOffsets;
    a.key_out = search ? ws + p.keys : nullptr;
    a.offsets = search ? nullptr : offsets;
    hipLaunchKernelGGL(group_small_kernel, dim3(1), dim3(kGroupThreads), 0, st, a, p.passes);
    HIP_TRY(hipGetLastError());
    return search ? launch_end(nullptr, nullptr, nullptr, 0, a.key_out, ws, nullptr, 0, offsets, E, st) : QINCO_OK;
  }
  unsigned long long* pairs = reinterpret_cast<unsigned long long*>(ws + p.pairs);
  int* went = reinterpret_cast<int*>(ws + p.went);
  const int bins = 1 << p.bits;
  const dim3 grid((unsigned)p.tiles), block(kGroupThreads);
  for (int pass = 0; pass < p.passes; ++pass) {
    a.shift = pass * p.bits;
    a.first = pass == 0;
    a.last = pass == p.passes - 1;
    a.pair_in = pass ? pairs + (int64_t)((pass - 1) & 1) * N : nullptr;
    a.pair_out = a.last ? nullptr : pairs + (int64_t)(pass & 1) * N;
    a.key_out = a.last && pass ? ws + p.keys : nullptr;
    a.start = a.last && pass ? ws + p.start : nullptr;
    a.went = pass ? went + (int64_t)(pass - 1) * N : nullptr;
    a.offsets = p.passes == 1 ? offsets : nullptr;
    with_ipt(p.ipt, [&](auto ipt) { hipLaunchKernelGGL((group_hist_kernel<decltype(ipt)::value>), grid, block, 0, st, a); });
    HIP_TRY(hipGetLastError());
    if (!a.tiles) {
      hipLaunchKernelGGL(group_scan_kernel, dim3((unsigned)((bins + 63) / 64)), dim3(1024), 0, st, a.counts, a.totals, (int)p.tiles, bins);
      HIP_TRY(hipGetLastError());
    }
    with_ipt(p.ipt, [&](auto ipt) { hipLaunchKernelGGL((group_scatter_kernel<decltype(ipt)::value>), grid, block, 0, st, a); });
    HIP_TRY(hipGetLastError());
  }
  if (p.passes == 1) return QINCO_OK;
  return launch_end(place, went, p.passes > 2 ? went + N : nullptr, N, a.key_out, ws, a.start, a.shift, offsets, E, st);
}

// rows of D elements, E of them a unit
static GroupRows group_rows_of(const int32_t* place, const int32_t* end, int64_t n, int32_t k, int64_t D, int E) {
  const int64_t units = (D + E - 1) / E;
  int l = 0;
  while (l < 6 && (1 << l) < units) ++l;
  return GroupRows{place, end, (long)n, (long)n * k, k, (int)D, (int)units, l};
}

// f(E): elements of type T in a unit of 16 bytes, or 1 for rows shorter than that
template <typename T, typename F>
static void with_unit(int64_t D, F f) {
  constexpr int E = 16 / sizeof(T);
  if (D >= E) f(std::integral_constant<int, E>{});
  else f(std::integral_constant<int, 1>{});
}

static dim3 group_grid(const GroupRows& g) {
  const long per = 256 >> g.lanes_log2;
  long b = (g.n + per - 1) / per;
  if (b > 65536) b = 65536;
  return dim3((unsigned)b);
}

extern "C" int qinco_group_gather(const void* x, int64_t x_stride_bytes, int64_t row_bytes, const int32_t* order, const int32_t* place,
                                  const int32_t* end, int64_t n, int32_t k, void* out, void* stream) {
  if (n < 0 || k < 1 || n > INT32_MAX / k || row_bytes < 1 || row_bytes > INT32_MAX || x_stride_bytes < 0)
    return fail(QINCO_ERR_INVALID, "qinco_group_gather: need n >= 0, k >= 1, n k < 2^31, 1 <= row_bytes < 2^31, a stride >= 0");
  if (n == 0) return QINCO_OK;
  if (!x || !order || !place || !end || !out) return fail(QINCO_ERR_INVALID, "qinco_group_gather: null buffer");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  auto go = [&](auto t) {
    using T = decltype(t);
    const int64_t D = row_bytes / (int64_t)sizeof(T);
    if (D == 1) {
      const GroupRows g = group_rows_of(place, end, n, k, 1, 1);
      const int64_t blocks = (g.N + 255) / 256;
      hipLaunchKernelGGL(group_pull_kernel<T>, dim3((unsigned)(blocks < (1 << 20) ? blocks : 1 << 20)), dim3(256), 0, st, g, order, (const T*)x,
                         (long)(x_stride_bytes / (int64_t)sizeof(T)), (T*)out);
      return;
    }
    with_unit<T>(D, [&](auto e) {
      constexpr int E = decltype(e)::value;
      const GroupRows g = group_rows_of(place, end, n, k, D, E);
      hipLaunchKernelGGL((group_gather_kernel<T, E>), group_grid(g), dim3(256), 0, st, g, (const T*)x,
                         (long)(x_stride_bytes / (int64_t)sizeof(T)), (T*)out);
    });
  };
  const uint64_t all = (uint64_t)row_bytes | (uint64_t)x_stride_bytes | reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out);
  if (all % 8 == 0) go(uint64_t{});
  else if (all % 4 == 0) go(uint32_t{});
  else if (all % 2 == 0) go(uint16_t{});
  else go(uint8_t{});
  HIP_TRY(hipGetLastError());
  return QINCO_OK;
}

template <typename F>
static void with_type(int dtype, F f) {
  if (dtype == QINCO_T_F32) f(float{});
  else if (dtype == QINCO_T_F16) f(_Float16{});
  else f(__bf16{});
}

static int check_rows(const char* who, int dtype, int w_dtype, bool weights, int64_t n, int32_t k, int32_t D) {
  if (!known(dtype)) return fail(QINCO_ERR_INVALID, "%s: unknown element type %d", who, dtype);
  if (weights && w_dtype != QINCO_T_F32 && w_dtype != dtype)
    return fail(QINCO_ERR_INVALID, "%s: weights are fp32 or of the rows' type", who);
  if (n < 0 || k < 1 || n > INT32_MAX / k || D < 1) return fail(QINCO_ERR_INVALID, "%s: need n >= 0, k >= 1, n k < 2^31, D >= 1", who);
  return QINCO_OK;
}

extern "C" int qinco_group_combine(const void* y, int dtype, int64_t y_stride, int32_t D, const void* weights, int w_dtype,
                                   const int32_t* place, int64_t n, int32_t k, void* out, void* stream) {
  if (int rc = check_rows("qinco_group_combine", dtype, w_dtype, weights != nullptr, n, k, D)) return rc;
  if (y_stride < 0) return fail(QINCO_ERR_INVALID, "qinco_group_combine: negative stride");
  if (n == 0) return QINCO_OK;
  if (!y || !place || !out) return fail(QINCO_ERR_INVALID, "qinco_group_combine: null buffer");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    with_unit<T>(D, [&](auto e) {
      constexpr int E = decltype(e)::value;
      const GroupRows g = group_rows_of(place, nullptr, n, k, D, E);
      // entries loaded together, 2 / 4 of them: 65536 rows of 2 x 768 bf16 64 / 75 us, 100000 of 3 x 32 8.0 / 9.4; 65536 of 8 x 128 fp32
      // 56 / 51, 4096 of 4 x 384 7.4 / 6.5
      if (k < 4) hipLaunchKernelGGL((group_combine_kernel<T, E, 2>), group_grid(g), dim3(256), 0, st, g, (const T*)y, (long)y_stride, weights, w_dtype, (T*)out);
      else hipLaunchKernelGGL((group_combine_kernel<T, E, 4>), group_grid(g), dim3(256), 0, st, g, (const T*)y, (long)y_stride, weights, w_dtype, (T*)out);
    });
  });
  HIP_TRY(hipGetLastError());
  return QINCO_OK;
}

extern "C" int qinco_group_combine_grad(const void* dout, int64_t dout_stride, const void* y, int64_t y_stride, int dtype, int32_t D,
                                        const void* weights, int w_dtype, const int32_t* place, const int32_t* end, int64_t n, int32_t k,
                                        void* dy, void* dw, void* stream) {
  if (int rc = check_rows("qinco_group_combine_grad", dtype, w_dtype, true, n, k, D)) return rc;
  if (y_stride < 0 || dout_stride < 0) return fail(QINCO_ERR_INVALID, "qinco_group_combine_grad: negative stride");
  if (n == 0) return QINCO_OK;
  if (!dout || !y || !weights || !place || !end || (!dy && !dw)) return fail(QINCO_ERR_INVALID, "qinco_group_combine_grad: null buffer");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  with_type(dtype, [&](auto t) {
    using T = decltype(t);
    auto go = [&](auto w) {
      using W = decltype(w);
      with_unit<T>(D, [&](auto e) {
        constexpr int E = decltype(e)::value;
        const GroupRows g = group_rows_of(place, end, n, k, D, E);
        hipLaunchKernelGGL((group_combine_grad_kernel<T, E, W>), group_grid(g), dim3(256), 0, st, g, (const T*)dout, (long)dout_stride,
                           (const T*)y, (long)y_stride, (const W*)weights, (T*)dy, (W*)dw);
      });
    };
    if (w_dtype == QINCO_T_F32) go(float{});
    else go(t);
  });
  HIP_TRY(hipGetLastError());
  return QINCO_OK;
}
