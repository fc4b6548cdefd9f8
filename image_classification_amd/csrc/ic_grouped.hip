// Products of rows with the matrix of their group, groups of ragged sizes.
//
//   group_rows   codes [n] -> order (the rows, group by group, ascending inside a group; rows of no
//                group last) and offsets (where each group begins in it)
//   forward      y_i  = W_g x_i            g = the group of row i, W [groups][out][k]
//   dx           dx_i = W_g^T dy_i
//   dw           dW_g = sum over the rows i of group g of dy_i x_i^T
//
// Nothing about the sizes of the groups is known on the host, and nothing is computed for it in a
// launch of its own.  Rows are cut into tiles of BM rows inside a group, and a workgroup finds its
// tile from the offsets alone: group e is given the tile numbers from floor(o_e / BM) + e on.
// These numbers ascend, and up to the next group's first there are
//     floor(o_{e+1} / BM) - floor(o_e / BM) + 1  >=  ceil((o_{e+1} - o_e) / BM)
// of them, so a grid of floor(n / BM) + groups + 1 tiles holds every tile of any ragged sizes; at
// most groups + 1 of its workgroups find nothing to do.  The last one or more tiles belong to the
// rows of no group, whose results are zeros.  A tile number's group is found by all 64 lanes of a
// wave at once, 64 offsets a step.
//
// The product itself: tiles of P rows x Q columns, 128 bytes of the contraction a stage, two
// stages in LDS filled by global_load_lds (16 bytes a lane straight into LDS, the next stage in
// flight while this one is multiplied), matrix instructions of 16 x 16 in float32 sums.  An operand
// whose contraction runs along its rows in memory is laid down as it is ([row][128 bytes]) and read
// 16 bytes a lane; one whose contraction runs across its rows ([contraction][columns]) is read by the
// transposing LDS load (16-bit types) or 4 bytes a lane (float32).  LDS-filling loads are linear in
// the lane, so the layouts are not padded: 16-byte granules are exchanged inside a row by an
// exclusive-or with bits of the row number, chosen so that the lanes of one LDS access fall into
// different banks.  Granules outside the operands are fetched from a granule of zeros.
#include <cmath>
#include <type_traits>

#include "ic_wave.h"

namespace ic {

namespace {

static __device__ __align__(16) const unsigned kZeroGranule[4] = {0u, 0u, 0u, 0u};

// ---- group_rows ----------------------------------------------------------------------------------
// A least-significant-digit radix sort of (group, row), digits of up to 9 bits, groups + 1 key values
// (the last one for rows of no group).  Equal digits keep their order: a wave takes 64 consecutive
// rows at a time and ranks them among the lanes of equal digit with one ballot per digit bit; the
// waves' counts are added in wave order.
constexpr int kMaxDigitBits = 9;

// The rank of this lane's digit among the 64 rows of the wave, on top of what cnt (this wave's counters)
// already holds; the counters go up.  Lanes that are not `in` hold no row.
template <typename Count>
__device__ __forceinline__ unsigned rank_in_wave(Count* cnt, unsigned d, bool in, int digit_bits,
                                                 unsigned long long below) {
  unsigned long long same = __ballot(in);
  for (int b = 0; b < digit_bits; ++b) {
    const unsigned long long ones = __ballot((d >> b) & 1u);
    same &= ((d >> b) & 1u) ? ones : ~ones;
  }
  // (only this wave touches its counters: lanes of equal digit read before the first one adds)
  const unsigned old = cnt[d];
  __builtin_amdgcn_wave_barrier();
  if (in && (same & below) == 0) cnt[d] = (Count)(old + __popcll(same));
  __builtin_amdgcn_wave_barrier();
  return old + __popcll(same & below);
}

// Few rows: one workgroup, everything in LDS.  Bound by latency: 6.6 us for 1000 rows of 1000 groups
// (bitonic sorting took 18.6 us: 66 steps of a barrier each), 4.0 for 16 rows of 64; up to 8192 rows of as many
// groups at most one such workgroup is about as fast as the launches below, or faster (5003 rows of 37 groups: 8.8 us
// against 23; 8192 rows of 8192 groups 25 against 24).  It also writes the offsets, with a search of the sorted keys
// for each, and that is what many more groups than rows cost: 1000 rows of 32 768 groups 30 us, of 2^20 730 (8193 rows
// of 2^20 groups, by the launches below: 45).
constexpr int kSmallRows = 8192, kSmallBits = 8;
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_group_small(const int32_t* __restrict__ codes, int n,
                                                         int64_t groups, int passes, int digit_bits,
                                                         int32_t* __restrict__ order,
                                                         int64_t* __restrict__ offsets) {
  constexpr int kWaves = THREADS / 64, kMost = THREADS == 1024 ? kSmallRows / THREADS : 1;
  constexpr int kRows = THREADS * kMost;
  __shared__ unsigned short cnt[kWaves][1 << kSmallBits];   // (at most 8192 rows)
  __shared__ unsigned keys[kRows];
  __shared__ unsigned short rows[kRows];
  __shared__ unsigned wave_sum[kWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int digits = 1 << digit_bits;
  const int rounds = (n + THREADS - 1) / THREADS;   // of 64 rows a wave
  const unsigned long long below = (1ull << lane) - 1ull;
  const int base = wave * 64 * rounds;
  unsigned key[kMost], row[kMost], rank[kMost];
#pragma unroll
  for (int r = 0; r < kMost; ++r) {
    const int i = base + r * 64 + lane;
    key[r] = 0;
    row[r] = (unsigned)i;
    if (r < rounds && i < n) {
      const int32_t c = codes[i];
      key[r] = c >= 0 && c < groups ? (unsigned)c : (unsigned)groups;
    }
  }
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * digit_bits;
    for (int d = lane; d < digits; d += 64) cnt[wave][d] = 0;
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int r = 0; r < kMost; ++r) {
      if (r >= rounds) break;
      const bool in = base + r * 64 + lane < n;
      const unsigned d = (key[r] >> shift) & (digits - 1);
      rank[r] = rank_in_wave(cnt[wave], d, in, digit_bits, below);
    }
    __syncthreads();
    // exclusive prefix over (digit, wave): thread d < digits sums its digit's waves
    unsigned total = 0;
    for (int d0 = 0; d0 < digits; d0 += THREADS) {
      const int d = d0 + (int)threadIdx.x;
      unsigned sum = 0;
      if (d < digits)
        for (int w = 0; w < kWaves; ++w) sum += cnt[w][d];
      unsigned inc = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned up = __shfl_up(inc, o, 64);
        if (lane >= o) inc += up;
      }
      if (lane == 63) wave_sum[wave] = inc;
      __syncthreads();
      unsigned run = total + inc - sum;
      for (int w = 0; w < kWaves; ++w) {
        const unsigned q = wave_sum[w];
        if (w < wave) run += q;
        total += q;
      }
      if (d < digits)
        for (int w = 0; w < kWaves; ++w) {
          const unsigned c = cnt[w][d];
          cnt[w][d] = (unsigned short)run;
          run += c;
        }
      __syncthreads();
    }
#pragma unroll
    for (int r = 0; r < kMost; ++r) {
      if (r >= rounds) break;
      if (base + r * 64 + lane < n) {
        const int at = cnt[wave][(key[r] >> shift) & (digits - 1)] + (int)rank[r];
        keys[at] = key[r];
        rows[at] = (unsigned short)row[r];
      }
    }
    __syncthreads();
    if (pass + 1 < passes) {
#pragma unroll
      for (int r = 0; r < kMost; ++r) {
        const int i = base + r * 64 + lane;
        if (r < rounds && i < n) {
          key[r] = keys[i];
          row[r] = rows[i];
        }
      }
      __syncthreads();
    }
  }
  for (int p = threadIdx.x; p < n; p += THREADS) order[p] = (int32_t)rows[p];
  for (int64_t e = threadIdx.x; e <= groups; e += THREADS) {   // the first position of a group >= e
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (keys[mid] < (unsigned)e) lo = mid + 1; else hi = mid;
    }
    offsets[e] = lo;
  }
}

// Many rows: a pass over a digit is three launches (counts per block of rows, prefixes, scatter).
// Bound by the launches' latency: 42 000 rows of 21 groups take 12.6 us in a captured graph, a million rows of
// 10 000 groups (two passes) 43, of which 12 MB read and written would be 5.
// A workgroup takes 4096 rows, or 2048 up to 2M rows, where a pass has few workgroups (42 000 rows 15.1 ->
// 12.6 us in a captured graph, 200 000 of 4000 groups 30 -> 25, 1M of 10 000 equal; 5M of 1000: 94 -> 104).
constexpr int64_t kSortFew = 2 << 20;
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
static_assert(kSortThreads >= 1 << kMaxDigitBits, "a thread holds the first place of a digit");

struct SortPlan {
  int bits;        // of the key: groups + 1 values, the last for rows of no group
  int passes;
  int digit_bits;
  int rows;        // of a workgroup
  int64_t blocks;
  size_t o_tab, o_total, o_pairs0, o_pairs1, o_codes, bytes;
};
SortPlan sort_plan(int64_t n, int64_t groups) {
  SortPlan p;
  p.bits = 1;
  while (((int64_t)1 << p.bits) < groups + 1) ++p.bits;
  p.passes = (p.bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (p.bits + p.passes - 1) / p.passes;
  p.rows = n <= kSortFew ? 2048 : 4096;
  p.blocks = (n + p.rows - 1) / p.rows;
  size_t off = 0;
  auto take = [&off](size_t b) {
    const size_t o = off;
    off += (b + 255) / 256 * 256;
    return o;
  };
  const size_t digits = (size_t)1 << p.digit_bits;
  p.o_tab = take(digits * p.blocks * 4);
  p.o_total = take(digits * 4);
  p.o_pairs0 = take(p.passes > 1 ? (size_t)n * 8 : 0);
  p.o_pairs1 = take(p.passes > 2 ? (size_t)n * 8 : 0);
  p.o_codes = take((size_t)n * 4);
  p.bytes = off;
  return p;
}

struct Pair {
  int32_t code, row;
};

__device__ __forceinline__ unsigned key_of(const int32_t* codes, const Pair* pairs, int64_t i,
                                           int64_t groups) {
  if (pairs) return (unsigned)pairs[i].code;
  const int32_t c = codes[i];
  return c >= 0 && c < groups ? (unsigned)c : (unsigned)groups;
}

// tab[digit][block] = rows of the block with that digit
template <int ROWS>
__global__ __launch_bounds__(kSortThreads) void k_sort_count(const int32_t* codes, const Pair* pairs,
                                                             int64_t n, int64_t groups, int shift,
                                                             int digit_bits, unsigned* tab) {
  __shared__ unsigned cnt[1 << kMaxDigitBits];
  const int digits = 1 << digit_bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * ROWS;
#pragma unroll
  for (int r = 0; r < ROWS / kSortThreads; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    if (i < n) atomicAdd(&cnt[(key_of(codes, pairs, i, groups) >> shift) & (digits - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) tab[(size_t)d * gridDim.x + blockIdx.x] = cnt[d];
}

// One workgroup a digit: its row of the table becomes an exclusive prefix, total[digit] the sum.
__global__ __launch_bounds__(256) void k_sort_scan(unsigned* tab, int64_t blocks, unsigned* total) {
  __shared__ unsigned part[256];
  unsigned* row = tab + (size_t)blockIdx.x * blocks;
  const int64_t b0 = blocks * threadIdx.x / 256, b1 = blocks * (threadIdx.x + 1) / 256;
  unsigned sum = 0;
  for (int64_t b = b0; b < b1; ++b) sum += row[b];
  part[threadIdx.x] = sum;
  __syncthreads();
  for (int o = 1; o < 256; o <<= 1) {
    const unsigned add = threadIdx.x >= (unsigned)o ? part[threadIdx.x - o] : 0;
    __syncthreads();
    part[threadIdx.x] += add;
    __syncthreads();
  }
  unsigned run = part[threadIdx.x] - sum;
  for (int64_t b = b0; b < b1; ++b) {
    const unsigned c = row[b];
    row[b] = run;
    run += c;
  }
  if (threadIdx.x == 255) total[blockIdx.x] = part[255];
}

// Rows to their places of this digit, keeping the order of equal digits: a wave takes 64
// consecutive rows at a time (rank among equal digits from ballots), the waves' counts are summed
// in wave order.
template <int ROWS>
__global__ __launch_bounds__(kSortThreads) void k_sort_scatter(
    const int32_t* codes, const Pair* pairs, int64_t n, int64_t groups, int shift, int digit_bits,
    const unsigned* tab, const unsigned* total, Pair* out_pairs, int32_t* out_order,
    int32_t* out_codes) {
  __shared__ unsigned cnt[kSortWaves][1 << kMaxDigitBits];
  __shared__ unsigned first[1 << kMaxDigitBits];
  __shared__ unsigned wave_sum[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int digits = 1 << digit_bits;
  for (int d = threadIdx.x; d < kSortWaves * digits; d += kSortThreads)
    cnt[d >> digit_bits][d & (digits - 1)] = 0;
  // exclusive prefix over the digits' totals (digits <= kSortThreads)
  unsigned v = threadIdx.x < (unsigned)digits ? total[threadIdx.x] : 0u;
  unsigned inc = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned up = __shfl_up(inc, o, 64);
    if (lane >= o) inc += up;
  }
  if (lane == 63) wave_sum[wave] = inc;
  __syncthreads();
  unsigned before = 0;
  for (int w = 0; w < wave; ++w) before += wave_sum[w];
  if (threadIdx.x < (unsigned)digits)
    first[threadIdx.x] = before + inc - v + tab[(size_t)threadIdx.x * gridDim.x + blockIdx.x];
  constexpr int kR = ROWS / kSortThreads;   // rounds of 64 rows a wave
  const int64_t base = (int64_t)blockIdx.x * ROWS + wave * (64 * kR);
  unsigned key[kR], rank[kR];
  const unsigned long long below = (1ull << lane) - 1ull;
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const int64_t i = base + r * 64 + lane;
    const bool in = i < n;
    key[r] = in ? key_of(codes, pairs, i, groups) : 0u;
    const unsigned d = (key[r] >> shift) & (digits - 1);
    rank[r] = rank_in_wave(cnt[wave], d, in, digit_bits, below);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < digits; d += kSortThreads) {
    unsigned run = first[d];
    for (int w = 0; w < kSortWaves; ++w) {
      const unsigned c = cnt[w][d];
      cnt[w][d] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const int64_t i = base + r * 64 + lane;
    if (i < n) {
      const unsigned d = (key[r] >> shift) & (digits - 1);
      const int64_t at = (int64_t)cnt[wave][d] + rank[r];
      const int32_t row = pairs ? pairs[i].row : (int32_t)i;
      if (out_pairs) {
        out_pairs[at] = Pair{(int32_t)key[r], row};
      } else {
        out_order[at] = row;
        out_codes[at] = (int32_t)key[r];
      }
    }
  }
}

// offsets[e] = first position whose group is >= e, from the sorted groups: the thread of a position
// where the group changes writes the offsets in between; a long run of empty groups is written by
// its wave.
__global__ __launch_bounds__(256) void k_group_offsets(const int32_t* sorted, int64_t n, int64_t groups,
                                                       int64_t* offsets) {
  const int lane = threadIdx.x & 63;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  int64_t e0 = 0, e1 = -1;   // offsets[e0 .. e1] = i
  if (i <= n) {
    e0 = i > 0 ? (int64_t)sorted[i - 1] + 1 : 0;
    e1 = i < n ? (int64_t)sorted[i] : groups;
    if (e1 > groups) e1 = groups;
  }
  const bool lots = e1 - e0 >= 16;
  if (!lots)
    for (int64_t e = e0; e <= e1; ++e) offsets[e] = i;
  unsigned long long who = __ballot(lots);
  while (who) {
    const int w = __ffsll(who) - 1;
    who &= who - 1;
    const int64_t a = __shfl(e0, w, 64), b = __shfl(e1, w, 64), at = __shfl(i, w, 64);
    for (int64_t e = a + lane; e <= b; e += 64) offsets[e] = at;
  }
}

// ---- finding a workgroup's tile --------------------------------------------------------------------
struct Groups {
  const int64_t* offsets;
  int64_t n, groups;
  // offsets as they are used: inside the rows, whatever the array holds
  __device__ __forceinline__ int64_t at(int64_t e) const {
    if (e <= 0) return 0;
    if (e > groups) return n;
    const int64_t o = offsets[e];
    return o < 0 ? 0 : o > n ? n : o;
  }
};

// A value that is the same in every lane, kept in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
  const unsigned low = __builtin_amdgcn_readfirstlane((unsigned)v);
  const unsigned high = __builtin_amdgcn_readfirstlane((unsigned)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)high << 32) | low);
}

// The last group e in [0, groups] whose first tile, at(e) / bm + e, is <= tile, and where its rows begin
// and end.  The 64 lanes of a wave look at 64 groups at a time, so that 63 groups take one round of
// loads and 10 000 take three; the last round's loads already hold the group's begin and end.
// (Four groups a lane are a round fewer and were slower: 40 groups apart, each lane's load is a cache
// line of its own.)
struct Found {
  int64_t e, o0, o1;
};
__device__ __forceinline__ Found find_group(const Groups& g, int64_t tile64, int64_t bm64, int lane) {
  // (rows, groups and tiles all fit 32 bits)
  const unsigned tile = (unsigned)tile64, bm = (unsigned)bm64, groups = (unsigned)g.groups;
  unsigned lo = 0, hi = groups + 1;
  for (;;) {
    const unsigned step = (hi - lo + 62u) / 63u;
    const unsigned e = lo + (unsigned)lane * step;
    const unsigned at = (unsigned)g.at(e < groups + 1 ? e : groups + 1);
    const int count = __popcll(__ballot(e < hi && at / bm + e <= tile));
    const int last = __builtin_amdgcn_readfirstlane(count > 0 ? count - 1 : 0);
    if (step == 1)
      return Found{(int64_t)(lo + (unsigned)last), (int64_t)(unsigned)__builtin_amdgcn_readlane((int)at, last),
                   (int64_t)(unsigned)__builtin_amdgcn_readlane((int)at, last + 1)};
    lo += (unsigned)last * step;
    hi = lo + step < hi ? lo + step : hi;
  }
}
// The same for a whole workgroup: its first wave looks (the others' loads of the same lines were a
// quarter of all loads where tiles are small), `box` [3] in LDS hands the answer on.
__device__ __forceinline__ Found find_group_once(const Groups& g, int64_t tile, int64_t bm, int wave, int lane,
                                                 unsigned* box) {
  if (wave == 0) {
    const Found f = find_group(g, tile, bm, lane);
    if (lane == 0) {
      box[0] = (unsigned)f.e;
      box[1] = (unsigned)f.o0;
      box[2] = (unsigned)f.o1;
    }
  }
  __syncthreads();
  return Found{(int64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)box[0]),
               (int64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)box[1]),
               (int64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)box[2])};
}

// Workgroup numbers are dealt to the 8 XCDs in turn; this gives each XCD a run of neighbours, whose
// tiles share rows or matrices in its L2.
__device__ __forceinline__ int64_t xcd_run(int64_t b, int64_t total) {
  const int64_t each = total / 8, rest = total % 8;
  const int64_t x = b & 7, i = b >> 3;
  return x * each + (x < rest ? x : rest) + i;
}

// ---- tiles in LDS ----------------------------------------------------------------------------------
constexpr int kStageBytes = 128;   // of the contraction

// 16 bytes a lane from memory to LDS at a wave-uniform address + 16 * lane.  Written as an instruction
// of its own, without results: the compiler, which cannot tell the stage being filled from the one
// being read by the transposing loads, would wait for it in front of every one of those.  The kernels
// wait themselves (all_landed) before the barrier that hands a stage over.
__device__ __forceinline__ void lds_load16(const void* src, char* lds_wave_base) {
  const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds_wave_base;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :
               : "v"(src), "s"(__builtin_amdgcn_readfirstlane(to))
               : "memory", "m0");
}
// The same from a scalar base and 32-bit offsets: no vector instruction besides the load itself.
__device__ __forceinline__ void lds_load16_at(const void* base, unsigned offset, char* lds_wave_base) {
  const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds_wave_base;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :
               : "v"(offset), "s"(base), "s"(__builtin_amdgcn_readfirstlane(to))
               : "memory", "m0");
}
__device__ __forceinline__ void lds_load4(const void* src, char* lds_wave_base) {
  const unsigned to = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)lds_wave_base;
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :
               : "v"(src), "s"(__builtin_amdgcn_readfirstlane(to))
               : "memory", "m0");
}
__device__ __forceinline__ void all_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// all but this wave's last COUNT loads
template <int COUNT>
__device__ __forceinline__ void all_but() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(COUNT) : "memory"); }

// Products of one granule of each operand (16 x 16 results).  float32 granules hold 4 elements, one
// product of depth 4 each (kParts): lane group g of element j stands for k = 4 g + j in both operands,
// and the order of k inside a step does not matter.  The products of one accumulator are kept apart by
// those of the others.
template <typename T> struct Mma;
template <> struct Mma<float> {
  static constexpr int kK = kStageBytes / 4, kParts = 4;
  static __device__ __forceinline__ f32x4 mul(int part, u32x4 q, u32x4 p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(q[part]), __uint_as_float(p[part]), c, 0, 0, 0);
  }
};
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <> struct Mma<bf16_t> {
  static constexpr int kK = kStageBytes / 2, kParts = 1;
  static __device__ __forceinline__ f32x4 mul(int, u32x4 q, u32x4 p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q),
                                                   __builtin_bit_cast(bf16x8, p), c, 0, 0, 0);
  }
};
template <> struct Mma<f16_t> {
  static constexpr int kK = kStageBytes / 2, kParts = 1;
  static __device__ __forceinline__ f32x4 mul(int, u32x4 q, u32x4 p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q),
                                                  __builtin_bit_cast(f16x8, p), c, 0, 0, 0);
  }
};

// Which columns the lanes of a fragment stand for.  A product of fragment j of the Q side leaves a lane
// with results 4 g .. 4 g + 3 of its 16, g = lane >> 4.  float32: result i of fragment j is column
// 16 j + i, so that the four lanes of a row store 64 neighbouring bytes an instruction.  16-bit types:
// column 8 (i >> 2) + 4 (j & 1) + (i & 3) + 32 (j >> 1), so that fragments 2 h and 2 h + 1 leave a lane with 8
// neighbouring columns and the four lanes store 64 neighbouring bytes as well.  (With 16 neighbouring
// columns a lane, whole lines of a row in four instructions of 16 bytes at a stride of 64, the stores
// of 1M x 64 float32 took 78 us of their own.)
template <typename T>
__device__ __forceinline__ constexpr int spread_row(int i) {   // of result i in fragment 0
  return sizeof(T) == 4 ? i : (i >> 2) * 8 + (i & 3);
}
template <typename T>
__device__ __forceinline__ constexpr int spread_step(int j) {  // from fragment 0 to fragment j
  return sizeof(T) == 4 ? j * 16 : (j & 1) * 4 + (j >> 1) * 32;
}

// Tile "along": [rows][128 bytes], granule s of row r holds granule s ^ swap(r) of the stage; 8 lanes
// of a read reach 8 different places of the 256 bytes of the banks.
__device__ __forceinline__ int along_swap_p(int r) { return r & 7; }
template <typename T>
__device__ __forceinline__ int along_swap_q(int r) {
  return sizeof(T) == 4 ? r & 7 : ((r >> 2) & 6) | ((r >> 1) & 1);
}
// A lane's place of fragment 0, step 0 (bytes behind the operand's tile).  Fragment i of P lies 16 i
// rows further, fragment j of Q spread_step(j) rows; step 1 exchanges the halves of a row (the swaps and the quarter
// wave's granule share no bit with it).
__device__ __forceinline__ int along_place_p(int r0, int lane) {
  const int r = r0 + (lane & 15);
  return r * kStageBytes + ((lane >> 4) ^ along_swap_p(r)) * 16;
}
template <typename T>
__device__ __forceinline__ int along_place_q(int r0, int lane) {
  const int r = r0 + spread_row<T>(lane & 15);
  return r * kStageBytes + ((lane >> 4) ^ along_swap_q<T>(r)) * 16;
}

// Tile "across": [kK rows of the contraction][COLS], granules exchanged by the contraction row k.  In
// the transposing load of 16-bit types the 16 lanes of a quarter wave point at 4 rows of the
// contraction and 4 x 4 columns; lane i is handed column i of the 16, 4 elements of the contraction.
// float32 needs no transposing: 4-byte loads of rows k, k + 1, ... a lane.
template <typename T, int COLS>
__device__ __forceinline__ int across_swap_p(int k) {
  if (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
  return COLS >= 128 ? ((k & 3) | ((k >> 1) & 4)) << 1 : (k & 3) << 1;
}
template <typename T, int COLS>
__device__ __forceinline__ int across_swap_q(int k) {
  if (sizeof(T) == 4) return ((k >> 2) & 3) << 2;
  return COLS >= 128 ? (k & 3) << 2 : (k & 1) << 2;
}
// A lane's place of fragment 0, step 0: the column whose 8 bytes (16-bit types) or 4 bytes (float32) it
// points at, in its row of the contraction.  The fragments' columns and the swaps only set bits that
// are clear in the wave's first column, so fragment i of P lies at place ^ 16 i columns and fragment j
// of Q at place ^ spread_step(j) columns; a step is kK / 2 rows.
template <typename T, int COLS, bool Q>
__device__ __forceinline__ int across_place(int c0, int lane) {
  constexpr int kRow = COLS * (int)sizeof(T), kV = 16 / (int)sizeof(T);
  const int k = sizeof(T) == 2 ? (lane >> 4) * 8 + ((lane & 15) >> 2) : (lane >> 4) * 4;
  int c;
  if (sizeof(T) == 2) c = (lane & 3) * (Q ? 8 : 4);
  else c = lane & 15;
  c += c0;
  const int swap = Q ? across_swap_q<T, COLS>(k) : across_swap_p<T, COLS>(k);
  return k * kRow + ((c / kV) ^ swap) * 16 + c % kV * (int)sizeof(T);
}
// (rows k .. k + 3 of float32 and k, k + 4 of the 16-bit types have the same swap)
template <typename T, int COLS>
__device__ __forceinline__ u32x4 read_across(const char* p) {
  constexpr int kRow = COLS * (int)sizeof(T);
  u32x4 out;
  if constexpr (sizeof(T) == 2) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(p));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s16x4*)(p + 4 * kRow));
    const u32x2 a = __builtin_bit_cast(u32x2, lo), b = __builtin_bit_cast(u32x2, hi);
    out[0] = a[0];
    out[1] = a[1];
    out[2] = b[0];
    out[3] = b[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = *reinterpret_cast<const unsigned*>(p + j * kRow);
  }
  return out;
}

// Reads the fragments of one operand for one step: COUNT of them from fragment `first` on.
template <typename T, int COLS, bool ALONG, bool Q, int COUNT>
__device__ __forceinline__ void read_fragments(const char* tile, int place, int step, int first, u32x4* out) {
  // (opaque: the fragments' addresses are worked out here, one instruction each, and not kept in
  // registers of their own through the loop)
  asm volatile("" : "+v"(place));
  if (ALONG) {
    const char* p = tile + (place ^ (step * 64));
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      out[i] = *reinterpret_cast<const u32x4*>(p + (Q ? spread_step<T>(first + i) : (first + i) * 16) * kStageBytes);
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i)
      out[i] = read_across<T, COLS>(tile + step * (Mma<T>::kK / 2 * COLS * (int)sizeof(T)) +
                                    (place ^ ((Q ? spread_step<T>(first + i) : (first + i) * 16) *
                                              (int)sizeof(T))));
  }
  __builtin_amdgcn_sched_barrier(0);
}

// One granule of an operand: elements [c, c + kVec) of a row of `cols` elements (NULL row: zeros), to
// LDS.  ALIGNED: granules begin at 16 bytes and do not cross the row's end.
template <typename T>
__device__ __forceinline__ u32x4 granule_of(const T* row, int64_t c, int64_t cols) {
  constexpr int kV = Elem<T>::kVec;
  u32x4 w = {0u, 0u, 0u, 0u};
  if (!row || c >= cols) return w;
  if (c + kV <= cols) {
    __builtin_memcpy(&w, row + c, 16);   // (a 16-byte load: memory may be read at any address)
  } else if (cols >= kV) {
    // the row's last granule, without what lies before c (element by element, the workgroups of a matrix's
    // last columns took several times as long as the others)
    u32x4 q;
    __builtin_memcpy(&q, row + cols - kV, 16);
    const unsigned drop = (unsigned)(c + kV - cols) * 8 * (unsigned)sizeof(T);   // bits, 16 to 112
    const uint64_t low = (uint64_t)q[1] << 32 | q[0], high = (uint64_t)q[3] << 32 | q[2];
    const uint64_t a = drop >= 64 ? high >> (drop - 64) : low >> drop | high << 1 << (63 - drop);
    const uint64_t b = drop >= 64 ? 0 : high >> drop;
    w = u32x4{(unsigned)a, (unsigned)(a >> 32), (unsigned)b, (unsigned)(b >> 32)};
  } else {
#pragma unroll
    for (int i = 0; i < kV; ++i)
      if (c + i < cols) {
        if constexpr (sizeof(T) == 2) {
          const unsigned b = reinterpret_cast<const unsigned short*>(row)[c + i];
          w[i >> 1] |= b << (16 * (i & 1));
        } else {
          w[i] = reinterpret_cast<const unsigned*>(row)[c + i];
        }
      }
  }
  return w;
}
template <typename T>
__device__ __forceinline__ void fetch(const T* row, int64_t c, int64_t cols, char* lds_wave_base) {
  const void* src = row && c < cols ? static_cast<const void*>(row + c)
                                    : static_cast<const void*>(kZeroGranule);
  lds_load16(src, lds_wave_base);
}

// The stages of a tile.  Each is multiplied in two steps, and a step in kHalves parts of the wave's
// rows (two where there are enough of them: the operands of half a step then fit the registers twice).
// A part's operands are read from LDS while the part before is multiplied, and the barrier that
// frees a stage's buffer stands in front of its last part, so that the matrix unit has work on both
// sides of it:
//     ... | read the last part | multiply the one before | stage st + 1 has landed, barrier |
//     read the first part of st + 1 | multiply the last part of st
// The freed buffer is refilled with stage st + 2 one load per four products, during the last part of
// st and (of four parts) the first of st + 1: issued in one go behind the barrier, the 8 waves' loads
// would hold up the products behind them in every wave.
// LOAD(i, stage, buffer) issues load i of kLoads (LOADS_EACH instructions) straight to the buffer; with
// PREPARES, NEXT(stage) fetches what the loads of that stage need, and lands a barrier before them.
#define MULTIPLY_STAGES(STAGES, LOAD, NEXT, PREPARES, LOADS_EACH)                     \
  {                                                                                  \
    constexpr int kStage = kPBytes + kQBytes;                                        \
    constexpr int kFirst = kHalves == 2 ? kLoads / 2 : kLoads;                       \
    auto none = [](int) {};                                                          \
    if (PREPARES) {                                                                  \
      NEXT(0);                                                                       \
      NEXT(1);                                                                       \
      all_landed();                                                                  \
      __syncthreads();                                                               \
    }                                                                                \
    _Pragma("unroll") for (int i = 0; i < kLoads; ++i) LOAD(i, 0, smem);             \
    if (STAGES > 1) {                                                                \
      _Pragma("unroll") for (int i = 0; i < kLoads; ++i) LOAD(i, 1, smem + kStage);  \
      all_but<kLoads * LOADS_EACH>();                                                \
    } else {                                                                         \
      all_landed();                                                                  \
    }                                                                                \
    __syncthreads();                                                                 \
    if (PREPARES) NEXT(2);                                                           \
    read_q(smem, 0, 0);                                                              \
    read_p(smem, 0, 0, 0);                                                           \
    for (int st = 0; st < STAGES; ++st) {                                            \
      char* buf = smem + (st & 1) * kStage;                                          \
      char* other = smem + ((st + 1) & 1) * kStage;                                  \
      if (kHalves == 2) {                                                            \
        read_p(buf, 0, 1, 1);                                                        \
      } else {                                                                       \
        read_q(buf, 1, 1);                                                           \
        read_p(buf, 1, 0, 1);                                                        \
      }                                                                              \
      const bool more = st > 0 && st + 1 < STAGES, refill = st + 2 < STAGES;         \
      mul(0, 0, 0, kLoads - kFirst, [&](int i) {                                     \
        if (more) LOAD(kFirst + i, st + 1, other);                                   \
      });                                                                            \
      if (PREPARES && st > 0) NEXT(st + 2);                                          \
      if (kHalves == 2) {                                                            \
        read_q(buf, 1, 1);                                                           \
        read_p(buf, 1, 0, 0);                                                        \
        mul(0, 1, 1, 0, none);                                                       \
        read_p(buf, 1, 1, 1);                                                        \
        mul(1, 0, 0, 0, none);                                                       \
      }                                                                              \
      all_landed();                                                                  \
      __syncthreads();                                                               \
      if (st + 1 < STAGES) {                                                         \
        read_q(other, 0, 0);                                                         \
        read_p(other, 0, 0, 0);                                                      \
      }                                                                              \
      constexpr int kLast = kHalves == 2 ? 1 : 0;                                    \
      mul(1, kLast, 1, kFirst, [&](int i) {                                          \
        if (refill) LOAD(i, st + 2, buf);                                            \
      });                                                                            \
    }                                                                                \
  }

// The same for operands of any alignment, which go through registers: LOAD(i, stage) fetches load i into
// them, PLACE(i, buffer) writes it to LDS a whole stage later, into the buffer that the barrier before has
// freed.
#define MULTIPLY_HELD(STAGES, LOAD, PLACE)                                           \
  {                                                                                  \
    constexpr int kStage = kPBytes + kQBytes;                                        \
    auto none = [](int) {};                                                          \
    _Pragma("unroll") for (int i = 0; i < kLoads; ++i) LOAD(i, 0);                   \
    _Pragma("unroll") for (int i = 0; i < kLoads; ++i) PLACE(i, smem);               \
    if (STAGES > 1) {                                                                \
      _Pragma("unroll") for (int i = 0; i < kLoads; ++i) LOAD(i, 1);                 \
    }                                                                                \
    __syncthreads();                                                                 \
    read_q(smem, 0, 0);                                                              \
    read_p(smem, 0, 0, 0);                                                           \
    for (int st = 0; st < STAGES; ++st) {                                            \
      char* buf = smem + (st & 1) * kStage;                                          \
      char* other = smem + ((st + 1) & 1) * kStage;                                  \
      if (kHalves == 2) {                                                            \
        read_p(buf, 0, 1, 1);                                                        \
      } else {                                                                       \
        read_q(buf, 1, 1);                                                           \
        read_p(buf, 1, 0, 1);                                                        \
      }                                                                              \
      mul(0, 0, 0, 0, none);                                                         \
      if (st + 1 < STAGES) {                                                         \
        _Pragma("unroll") for (int i = 0; i < kLoads; ++i) PLACE(i, other);          \
      }                                                                              \
      if (st + 2 < STAGES) {                                                         \
        _Pragma("unroll") for (int i = 0; i < kLoads; ++i) LOAD(i, st + 2);          \
      }                                                                              \
      if (kHalves == 2) {                                                            \
        read_q(buf, 1, 1);                                                           \
        read_p(buf, 1, 0, 0);                                                        \
        mul(0, 1, 1, 0, none);                                                       \
        read_p(buf, 1, 1, 1);                                                        \
        mul(1, 0, 0, 0, none);                                                       \
      }                                                                              \
      __syncthreads();                                                               \
      if (st + 1 < STAGES) {                                                         \
        read_q(other, 0, 0);                                                         \
        read_p(other, 0, 0, 0);                                                      \
      }                                                                              \
      constexpr int kLast = kHalves == 2 ? 1 : 0;                                    \
      mul(1, kLast, 1, 0, none);                                                     \
    }                                                                                \
  }

struct RowsArgs {
  const void* p;       // rows [n][ld_p], contraction along
  const void* q;       // matrices [groups][...]
  void* y;
  Groups g;
  const int32_t* order;
  int64_t ld_p, ld_q, ld_y, q_stride;
  int depth;           // length of the contraction
  int cols;            // columns of the result
  int col_tiles;
  int y_f32;
  int64_t id0;         // the first tile of this launch
};

// A lane's sixteen results of one row, v[j] those of fragment j, in the 64 columns from c on; the row
// begins at `at` and has `cols` columns.  vec: 16 bytes can be stored at once.
template <typename T>
__device__ __forceinline__ void store16(void* y, int64_t at, int c, int cols, int lane, bool f32, const f32x4* v) {
  if (sizeof(T) == 4 || f32) {
    float* d = static_cast<float*>(y) + at;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int cj = c + spread_row<T>((lane >> 4) * 4) + spread_step<T>(j);
      if (cj + 4 <= cols) {
        __builtin_memcpy(d + cj, &v[j], 16);     // (a 16-byte store: memory may be written at any address)
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (cj + i < cols) d[cj + i] = v[j][i];
      }
    }
  } else if constexpr (sizeof(T) == 2) {
    T* d = static_cast<T*>(y) + at;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int cj = c + spread_row<T>((lane >> 4) * 4) + spread_step<T>(2 * h);
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v[2 * h + (i >> 2)][i & 3];
      if (cj + 8 <= cols) {
        const u32x4 w = Elem<T>::pack(f);
        __builtin_memcpy(d + cj, &w, 16);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (cj + i < cols) Elem<T>::store(d + cj + i, f[i]);
      }
    }
  }
}

// forward (QALONG: W_g [cols][depth]) and dx (W_g [depth][cols])
// 65 536 rows, 16 groups of 2048 x 2048 bf16, 256 x 256 tiles: 592 us forward and 611 dx, 930 and 900
// TFLOP/s (a large library product reaches 1280).  The products alone, with neither loads nor LDS reads,
// take 440 us (the clock falls to about 2.2 GHz under them, and some 2100 tiles make 9 rounds of 256 CUs
// where 8.2 would do); the LDS reads cost 80 us more, the loads as much again.
// 42 000 rows, 21 groups, 1000 -> 256 float32: 237 us forward (64 x 64 tiles) and 243 dx (128 x 128), 90
// TFLOP/s where a large library product reaches 154; the products alone 190 and 220 us, because 2.6 and
// 5.5 rounds of the card take 3 and 6.
// Rows that are not 16-byte pieces (ALIGNED false): 5003 rows, 37 groups, 193 -> 317 fp16 10.4 and 10.8 us, 24 340 rows,
// 3 groups, 423 -> 1566 fp16 96 us forward and 151 dx (of 424 -> 1568 columns 68 and 60): bound by the
// instructions that put their pieces together.
template <typename T, int BM, int BN, int WM, int WN, bool QALONG, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_grouped_rows(RowsArgs a) {
  constexpr int kThreads = WM * WN * 64, kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static_assert(FN == 4, "64 columns a wave");
  constexpr int kV = Elem<T>::kVec, kK = Mma<T>::kK;
  constexpr int kPBytes = BM * kStageBytes, kQBytes = BN * kStageBytes;
  constexpr int kPLoads = BM * 8 / kThreads, kQLoads = BN * 8 / kThreads;
  constexpr int kQRow = BN * (int)sizeof(T) / 16;   // granules of a contraction row (across)
  static_assert(kPLoads * kThreads == BM * 8 && kQLoads * kThreads == BN * 8, "tile");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int* rows = reinterpret_cast<int*>(smem + 2 * (kPBytes + kQBytes));
  __shared__ unsigned box[3];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = a.id0 + xcd_run(blockIdx.x, gridDim.x);
  const int64_t tile = id / a.col_tiles;
  const int c0 = (int)(id % a.col_tiles) * BN;
  const Found f = find_group_once(a.g, tile, BM, wave, lane, box);
  const int64_t e = f.e, o0 = f.o0, o1 = f.o1;
  const int64_t t = tile - (o0 / BM + e);
  const int64_t r0 = o0 + t * BM;
  if (t < 0 || r0 >= o1) return;   // (t < 0: only if the offsets do not ascend)
  const int m = o1 - r0 < BM ? (int)(o1 - r0) : BM;
  // the number of a row of the tile; -1 behind the group's end and for an entry of `order` that is no row
  auto row_at = [&](int i) {
    if (i >= m) return (int64_t)-1;
    const int64_t r = a.order ? (int64_t)a.order[r0 + i] : r0 + i;
    return r >= 0 && r < a.g.n ? r : (int64_t)-1;
  };
  const int wm = wave % WM, wn = wave / WM;
  const int pr = wm * (BM / WM), qc = wn * (BN / WN);
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // (for the end; read behind the barriers of the stages)
  for (int i = threadIdx.x; i < BM; i += kThreads) rows[i] = (int)row_at(i);

  if (e < a.g.groups) {
    const T* qb = static_cast<const T*>(a.q) + e * a.q_stride;
    // P: the rows of this lane's granules (behind the group's end row 0 stands in: such rows are
    // multiplied and not stored)
    const int lin = wave * 64 + lane;
    const int along = ((lin & 7) ^ along_swap_p(lin >> 3)) * kV;   // (a step of i keeps the low bits)
    const T* prow[kPLoads];
#pragma unroll
    for (int i = 0; i < kPLoads; ++i) {
      const int64_t row = row_at(((i * kWaves + wave) * 64 + lane) >> 3);
      prow[i] = static_cast<const T*>(a.p) + (row < 0 ? 0 : row) * a.ld_p;
    }
    // Q: granule i of this lane lies kQStep rows of the matrix behind granule 0.  Where the tile lies
    // inside the matrix, a load is a scalar base and one of (at most) two offsets that a lane keeps.
    constexpr int kQStep = QALONG ? kThreads / 8 : kThreads / kQRow;
    const int qfirst = QALONG ? lin >> 3 : lin / kQRow;
    auto qgranule = [&](int i) {
      return QALONG ? (lin & 7) ^ along_swap_q<T>(qfirst + i * kQStep)
                    : (lin % kQRow) ^ across_swap_q<T, BN>(qfirst + i * kQStep);
    };
    const unsigned qoff0 = (unsigned)(qfirst * a.ld_q + qgranule(0) * kV) * (unsigned)sizeof(T);
    const unsigned qoff1 = (unsigned)(qfirst * a.ld_q + qgranule(1) * kV) * (unsigned)sizeof(T);
    const bool inside = ALIGNED && c0 + BN <= a.cols;
    const int full = a.depth / kK;     // stages that lie inside the depth
    constexpr int kLoads = kPLoads + kQLoads;
    u32x4 held[ALIGNED ? 1 : kLoads];
    auto load = [&](int i, int st, char* buf) {
      const int64_t k0 = (int64_t)st * kK;
      if (i < kPLoads) {
        char* to = buf + (i * kWaves + wave) * 1024;
        if constexpr (!ALIGNED) held[i] = granule_of<T>(prow[i], k0 + along, a.depth);
        else if (st < full) lds_load16(prow[i] + along + k0, to);
        else fetch<T>(prow[i], k0 + along, a.depth, to);
        return;
      }
      const int q = i - kPLoads;
      char* to = buf + kPBytes + (q * kWaves + wave) * 1024;
      if (inside && st < full) {
        const T* base = QALONG ? qb + (int64_t)(c0 + q * kQStep) * a.ld_q + k0 : qb + (k0 + q * kQStep) * a.ld_q + c0;
        if constexpr (ALIGNED) lds_load16_at(base, q % 2 ? qoff1 : qoff0, to);
        return;
      }
      const T* row;
      int64_t from, width;
      if (QALONG) {
        const int c = c0 + qfirst + q * kQStep;
        row = c < a.cols ? qb + (int64_t)c * a.ld_q : nullptr;
        from = k0 + qgranule(q) * kV;
        width = a.depth;
      } else {
        const int64_t k = k0 + qfirst + q * kQStep;
        row = k < a.depth ? qb + k * a.ld_q : nullptr;
        from = c0 + qgranule(q) * kV;
        width = a.cols;
      }
      if constexpr (ALIGNED) fetch<T>(row, from, width, to);
      else held[i] = granule_of<T>(row, from, width);
    };
    auto place = [&](int i, char* buf) {
      if constexpr (!ALIGNED) {
        char* to = i < kPLoads ? buf + (i * kWaves + wave) * 1024
                               : buf + kPBytes + ((i - kPLoads) * kWaves + wave) * 1024;
        *reinterpret_cast<u32x4*>(to + lane * 16) = held[i];
      }
    };
    const int stages = (int)(((int64_t)a.depth + kK - 1) / kK);
    const bool busy = pr < m;   // a wave whose rows all lie behind the group's end only loads
    constexpr int kHalves = FM >= 4 ? 2 : 1, kHalf = FM / kHalves;
    u32x4 pf[2][kHalf], qf[2][FN];
    const int pplace = along_place_p(pr, lane);
    const int qplace = kPBytes + (QALONG ? along_place_q<T>(qc, lane) : across_place<T, BN, true>(qc, lane));
    auto read_p = [&](const char* buf, int step, int half, int to) {
      if (busy) read_fragments<T, BM, true, false, kHalf>(buf, pplace, step, half * kHalf, pf[to]);
    };
    auto read_q = [&](const char* buf, int step, int to) {
      if (busy) read_fragments<T, BN, QALONG, true, FN>(buf, qplace, step, 0, qf[to]);
    };
    // `count` loads are issued between the products
    auto mul = [&](int q, int half, int p, int count, auto&& issue) {
#pragma unroll
      for (int i = 0; i < kHalf; ++i) {
        if (busy)
#pragma unroll
        for (int part = 0; part < Mma<T>::kParts; ++part)
#pragma unroll
          for (int j = 0; j < FN; ++j)
            acc[half * kHalf + i][j] = Mma<T>::mul(part, qf[q][j], pf[p][i], acc[half * kHalf + i][j]);
        if (count > 0) {
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int l = 0; l < kLoads; ++l)
            if (l < count && l * kHalf / count == i) issue(l);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    };
    auto next = [](int) {};
    if constexpr (ALIGNED) {
      MULTIPLY_STAGES(stages, load, next, false, 1)
    } else {
      auto fill = [&](int i, int st) { load(i, st, smem); };
      MULTIPLY_HELD(stages, fill, place)
    }
  } else {
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int row = rows[pr + i * 16 + (lane & 15)];
    if (row >= 0) store16<T>(a.y, (int64_t)row * a.ld_y, c0 + qc, a.cols, lane, a.y_f32, acc[i]);
  }
}

// Short rows (a contraction of at most NS stages, 512 bytes: the 128 float32 of a local descriptor), tiles
// of 64 R x 64: there are too few stages to pipeline, so everything is fetched at once.  The matrix's part
// goes to LDS, shared by the four waves; each wave's 16 R rows go straight to the registers that the
// products take them from.  One barrier, one memory latency behind the search for the group.
// 1M rows x 128 float32, 10 000 groups of 64 x 128: 301 us in a captured graph, 3.7 TB/s of rows, matrices and results and
// 54 TFLOP/s (310 to 337 under a kernel trace, where R = 1 takes 343 and staging like the longer ones 355).  Neither is at its limit (memory 0.21 ms, products
// 0.11 ms): a workgroup loads, multiplies and stores once, and what four of them a CU overlap is part
// of it.
// Five workgroups share a CU (R = 2: four): 32 KB of LDS and 96 (128) registers each.
template <typename T, int NS, int R, bool QALONG>
__global__ __launch_bounds__(256, R == 1 ? 5 : 3) void k_grouped_short(RowsArgs a) {
  constexpr int BN = 64, kWaves = 4, FN = 4, BM = 64 * R;
  constexpr int kV = Elem<T>::kVec, kK = Mma<T>::kK;
  constexpr int kQRow = BN * (int)sizeof(T) / 16;
  constexpr int kStage = BN * kStageBytes;
  __shared__ __attribute__((aligned(1024))) char smem[NS * kStage];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = a.id0 + xcd_run(blockIdx.x, gridDim.x);
  const int64_t tile = id / a.col_tiles;
  const int c0 = (int)(id % a.col_tiles) * BN;
  // (what still loads goes before what multiplies: 3 %)
  __builtin_amdgcn_s_setprio(3);
  const Found f = find_group_once(a.g, tile, BM, wave, lane, reinterpret_cast<unsigned*>(smem));
  __syncthreads();   // (the box is read: its place may be filled)
  const int64_t t = tile - (f.o0 / BM + f.e);
  const int64_t r0 = f.o0 + t * BM;
  if (t < 0 || r0 >= f.o1) return;
  // the last tile of a group leaves waves without rows: not the same ones in every tile
  const int quarter = (wave + (int)tile) & 3;
  int64_t row[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t pos = r0 + (r * 4 + quarter) * 16 + (lane & 15);
    row[r] = -1;
    if (pos < f.o1) {
      row[r] = a.order ? (int64_t)a.order[pos] : pos;
      if (row[r] < 0 || row[r] >= a.g.n) row[r] = -1;
    }
  }
  f32x4 acc[R][FN];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[r][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (f.e < a.g.groups) {
    u32x4 pf[R][2 * NS];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const bool busy = r0 + (r * 4 + quarter) * 16 < f.o1;
      const T* p = static_cast<const T*>(a.p) + (row[r] < 0 ? 0 : row[r]) * a.ld_p + (lane >> 4) * kV;
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        const int k = i * 4 * kV;
        pf[r][i] = busy && k + (lane >> 4) * kV < a.depth ? *reinterpret_cast<const u32x4*>(p + k)
                                                          : u32x4{0u, 0u, 0u, 0u};
      }
    }
    const T* qb = static_cast<const T*>(a.q) + f.e * a.q_stride;
    const int lin = wave * 64 + lane;
#pragma unroll
    for (int st = 0; st < NS; ++st)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int q = i * 256 + lin;
        char* to = smem + st * kStage + (i * kWaves + wave) * 1024;
        if (QALONG) {
          const int r = q >> 3;
          fetch<T>(c0 + r < a.cols ? qb + (int64_t)(c0 + r) * a.ld_q : nullptr,
                         st * kK + ((q & 7) ^ along_swap_q<T>(r)) * kV, a.depth, to);
        } else {
          const int k = q / kQRow;
          fetch<T>(st * kK + k < a.depth ? qb + (int64_t)(st * kK + k) * a.ld_q : nullptr,
                         c0 + ((q % kQRow) ^ across_swap_q<T, BN>(k)) * kV, a.cols, to);
        }
      }
    const int qplace = QALONG ? along_place_q<T>(0, lane) : across_place<T, BN, true>(0, lane);
    all_landed();
    __syncthreads();
    __builtin_amdgcn_s_setprio(0);
    const bool busy = r0 + quarter * 16 < f.o1, second = R > 1 && r0 + (4 + quarter) * 16 < f.o1;
    if (busy) {
#pragma unroll
      for (int i = 0; i < 2 * NS; ++i) {
        u32x4 qf[FN];
        read_fragments<T, BN, QALONG, true, FN>(smem + i / 2 * kStage, qplace, i % 2, 0, qf);
#pragma unroll
        for (int part = 0; part < Mma<T>::kParts; ++part)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[0][j] = Mma<T>::mul(part, qf[j], pf[0][i], acc[0][j]);
        if constexpr (R > 1) {
          if (second)
#pragma unroll
            for (int part = 0; part < Mma<T>::kParts; ++part)
#pragma unroll
              for (int j = 0; j < FN; ++j) acc[R - 1][j] = Mma<T>::mul(part, qf[j], pf[R - 1][i], acc[R - 1][j]);
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (row[r] >= 0) store16<T>(a.y, row[r] * a.ld_y, c0, a.cols, lane, a.y_f32, acc[r]);
}

// Few rows a group (single rows to serve): the matrices are the traffic, so a workgroup takes 16 rows
// of a group and few columns and keeps as many loads in flight as its registers hold; nothing is
// shared, so nothing goes through LDS on the way.  BYDEPTH: the four waves share the depth of the same
// 32 columns and add their sums in LDS, in wave order; otherwise (short rows) each wave takes 16 columns
// of its own.  A lane's granules of a chunk are neighbours (32 bytes), four lanes read 128 bytes.
// 16 rows, 64 groups of 2048 x 2048 bf16 (about 14 of them met, 118 MB): 27.5 us, 4.3 TB/s (through LDS 36 us);
// 1000 rows, 1000 groups of 64 x 128 float32 (21 MB): 10.6 us.
// QALONG false (dx of float32, by depth only): the matrix's granules are gathered from four of its rows, 16
// neighbouring columns a load; for launches that latency bounds (18 rows, 3 groups of 1336 x 184: 39.6 -> 13.4
// us; 128 rows, 1 group of 1024 x 1024: 30.5 -> 10.1).
template <typename T, bool BYDEPTH, bool QALONG, bool ALIGNED>
__global__ __launch_bounds__(256) void k_grouped_few(RowsArgs a) {
  constexpr int kV = Elem<T>::kVec;
  constexpr int kChunk = 8 * kV;                 // of the depth: 2 granules in each quarter wave
  constexpr int CF = BYDEPTH ? 2 : 1;            // fragments of 16 columns a wave
  constexpr int kCols = BYDEPTH ? 32 : 64;       // of a workgroup
  static_assert(QALONG || (BYDEPTH && sizeof(T) == 4), "dx: float32 by depth");
  constexpr int kAhead = BYDEPTH ? 4 : 2;        // chunks whose loads are in flight together
  __shared__ f32x4 sums[BYDEPTH ? 4 : 1][CF][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = a.id0 + blockIdx.x;
  const int64_t tile = id / a.col_tiles;
  const int c0 = (int)(id % a.col_tiles) * kCols + (BYDEPTH ? 0 : wave * 16);
  __shared__ unsigned box[3];
  const Found f = find_group_once(a.g, tile, 16, wave, lane, box);
  const int64_t e = f.e, o0 = f.o0, o1 = f.o1;
  const int64_t t = tile - (o0 / 16 + e);
  const int64_t r0 = o0 + t * 16;
  if (t < 0 || r0 >= o1) return;
  int64_t row = -1;
  if (r0 + (lane & 15) < o1) {
    row = a.order ? (int64_t)a.order[r0 + (lane & 15)] : r0 + (lane & 15);
    if (row < 0 || row >= a.g.n) row = -1;
  }
  f32x4 acc[CF];
#pragma unroll
  for (int j = 0; j < CF; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
  if (e < a.g.groups) {
    const int kq = (lane >> 4) * 2 * kV;
    const T* p = static_cast<const T*>(a.p) + (row < 0 ? 0 : row) * a.ld_p + kq;
    const T* q[CF];
#pragma unroll
    for (int j = 0; j < CF; ++j) {
      int c = c0 + j * 16 + (lane & 15);
      if (c >= a.cols) c = a.cols - 1;           // (its products are not stored)
      q[j] = static_cast<const T*>(a.q) + e * a.q_stride + (QALONG ? (int64_t)c * a.ld_q + kq : (int64_t)c);
    }
    // four elements of a column from row k on
    auto across = [&](const T* col, int k) {
      u32x4 w = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (k + i < a.depth) w[i & 3] = *reinterpret_cast<const unsigned*>(col + (int64_t)(k + i) * a.ld_q);
      return w;
    };
    const int chunks = (a.depth + kChunk - 1) / kChunk;
    const int first = BYDEPTH ? (int)((int64_t)chunks * wave / 4) : 0;
    const int last = BYDEPTH ? (int)((int64_t)chunks * (wave + 1) / 4) : chunks;
    for (int c = first; c < last; c += kAhead) {
      u32x4 pv[kAhead][2], qv[kAhead][CF][2];
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = (c + i) * kChunk + h * kV;
          if constexpr (!QALONG) {
            const bool in = c + i < last;
            pv[i][h] = granule_of<T>(p, k, in ? a.depth - kq : 0);
#pragma unroll
            for (int j = 0; j < CF; ++j) qv[i][j][h] = across(q[j], in ? k + kq : a.depth);
          } else if constexpr (ALIGNED) {
            const bool in = c + i < last && k + kq < a.depth;
            pv[i][h] = in ? *reinterpret_cast<const u32x4*>(p + k) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
            for (int j = 0; j < CF; ++j)
              qv[i][j][h] = in ? *reinterpret_cast<const u32x4*>(q[j] + k) : u32x4{0u, 0u, 0u, 0u};
          } else {
            const int width = c + i < last ? a.depth - kq : 0;    // of what begins at this lane's pointers
            pv[i][h] = granule_of<T>(p, k, width);
#pragma unroll
            for (int j = 0; j < CF; ++j) qv[i][j][h] = granule_of<T>(q[j], k, width);
          }
        }
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int part = 0; part < Mma<T>::kParts; ++part)
#pragma unroll
            for (int j = 0; j < CF; ++j) acc[j] = Mma<T>::mul(part, qv[i][j][h], pv[i][h], acc[j]);
    }
  }
  if (BYDEPTH) {
#pragma unroll
    for (int j = 0; j < CF; ++j) sums[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= CF) return;
    // wave j finishes fragment j
    acc[0] = sums[0][wave][lane];
#pragma unroll
    for (int w = 1; w < 4; ++w) acc[0] += sums[w][wave][lane];
  }
  const int c = c0 + (BYDEPTH ? wave * 16 : 0) + (lane >> 4) * 4;
  if (row < 0) return;
  const int64_t at = row * a.ld_y + c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < a.cols) {
      if (a.y_f32 || sizeof(T) == 4) static_cast<float*>(a.y)[at + i] = acc[0][i];
      else Elem<T>::store(static_cast<T*>(a.y) + at + i, acc[0][i]);
    }
}

// ---- dw ---------------------------------------------------------------------------------------------
// dW_e[o][k] = sum_r dy[r][o] x[r][k]: both operands run across the contraction, whose length, the
// group's rows, is ragged.  All the work is one line of units: group after group, for each tile of
// its matrix the stages of its rows; a group has floor(o_{e+1} / kK) + 1 - floor(o_e / kK) stages in it
// (at least as many as it needs, at least one, at most one too many), so that the place of any unit
// follows from the offsets as for the row tiles above.  The launch's workgroups (as many as fit the
// card at a time) each take an equal run of the line.  A tile whose stages all fall into one run is
// stored at once; the pieces of one that is cut go to float32 partial results -- at most two a
// workgroup: of the tile its run begins inside (number 2 w) and of the one it ends inside (2 w + 1) --
// and k_grouped_dw_join adds them in the order of the line.
// 65 536 rows, 16 groups of 2048 x 2048 bf16: 721 us and 46 to join, 720 TFLOP/s together; without loads
// 510 us, without LDS reads either 475.  42 000 rows, 21 groups of 256 x 1000 float32: 236 + 21 us.  5003 rows,
// 37 groups of 317 x 193 fp16: 18 + 9 us.
struct DwArgs {
  const void* dy;
  const void* x;
  void* dw;
  float* part;
  Groups g;
  const int32_t* order;
  int64_t ld_dy, ld_x;
  int out, k;
  int tiles, k_tiles;
  int wgs;
  int whole;           // runs begin and end with tiles
  int y_f32;
};

// A place in the line.
struct DwPlace {
  int64_t e, o0, o1;   // the group and its rows
  int tile;            // of its matrix
  int64_t stage, stages;   // the stage, and how many the line has for each tile of the group
};
__device__ __forceinline__ int64_t dw_line(const DwArgs& a, int64_t kk) {
  return (uniform(a.g.at(a.g.groups)) / kk + a.g.groups) * a.tiles;
}
__device__ __forceinline__ DwPlace dw_place(const DwArgs& a, int64_t u, int64_t kk, int lane) {
  DwPlace p;
  const Found f = find_group(a.g, u / a.tiles, kk, lane);
  p.e = f.e < a.g.groups ? f.e : a.g.groups - 1;   // (it always is if the offsets ascend)
  p.o0 = f.o0;
  p.o1 = f.o1;
  if (p.o1 < p.o0) p.o1 = p.o0;
  p.stages = p.o1 / kk + 1 - p.o0 / kk;
  int64_t in = u - (p.o0 / kk + p.e) * a.tiles;
  if (in < 0) in = 0;
  const int64_t t = in / p.stages;
  p.tile = t < a.tiles ? (int)t : a.tiles - 1;
  p.stage = in % p.stages;
  return p;
}

// From a place to the first stage of the next tile, without a search; false behind the last group.
__device__ __forceinline__ bool dw_next(const DwArgs& a, DwPlace& p, int64_t kk) {
  p.stage = 0;
  if (++p.tile < a.tiles) return true;
  p.tile = 0;
  if (++p.e >= a.g.groups) return false;
  p.o0 = uniform(a.g.at(p.e));
  p.o1 = uniform(a.g.at(p.e + 1));
  if (p.o1 < p.o0) p.o1 = p.o0;
  p.stages = p.o1 / kk + 1 - p.o0 / kk;
  return true;
}

// The unit that workgroup w's run begins with (and w - 1's ends before).  Whole tiles: the first unit of a
// tile, an equal number of tiles each.
__device__ __forceinline__ int64_t dw_begin(const DwArgs& a, int64_t line, int64_t w, int64_t kk) {
  if (!a.whole) return line * w / a.wgs;
  const int64_t t = a.g.groups * a.tiles * w / a.wgs, e = t / a.tiles;
  if (e >= a.g.groups) return line;
  const int64_t o0 = uniform(a.g.at(e)), o1 = uniform(a.g.at(e + 1));
  const int64_t stages = (o1 < o0 ? o0 : o1) / kk + 1 - o0 / kk;
  return (o0 / kk + e) * a.tiles + t % a.tiles * stages;
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_grouped_dw(DwArgs a) {
  constexpr int kThreads = WM * WN * 64, kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  static_assert(FN == 4, "64 columns a wave");
  static_assert(BM == BN, "both operands' granules lie in the same rows");
  constexpr int kV = Elem<T>::kVec, kK = Mma<T>::kK;
  constexpr int kPBytes = BM * kStageBytes, kQBytes = BN * kStageBytes;
  constexpr int kPLoads = BM * 8 / kThreads;
  constexpr int kPRow = BM * (int)sizeof(T) / 16;   // granules of a contraction row
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // neighbours in the line share rows: they run on one XCD
  const int64_t w = xcd_run(blockIdx.x, gridDim.x);
  const int64_t line = dw_line(a, kK);
  int64_t u = dw_begin(a, line, w, kK);
  const int64_t u1 = dw_begin(a, line, w + 1, kK);
  const int wm = wave % WM, wn = wave / WM;
  const int pc = wm * (BM / WM), qc = wn * (BN / WN);
  const int pplace = across_place<T, BM, false>(pc, lane);
  const int qplace = kPBytes + across_place<T, BN, true>(qc, lane);
  int* ids = reinterpret_cast<int*>(smem + 2 * (kPBytes + kQBytes));   // [2][kK] rows of a stage
  if (u >= u1) return;
  DwPlace pl = dw_place(a, u, kK, lane);
  for (int64_t done = 0;;) {
    const int64_t run = pl.stages - pl.stage < u1 - u ? pl.stages - pl.stage : u1 - u;
    u += run;
    const int m0 = pl.tile / a.k_tiles * BM, n0 = pl.tile % a.k_tiles * BN;
    const int64_t r0 = pl.o0 + pl.stage * kK;
    int64_t r1 = r0 + run * kK;
    if (r1 > pl.o1) r1 = pl.o1;
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (r0 < r1) {
      // The rows of a stage: `order` goes to LDS, one wave's load a stage, two stages ahead of the
      // loads that need it (without an order the positions are the rows).
      const int64_t stages = (r1 - r0 + kK - 1) / kK;
      // this lane's first granule of either operand, and its row stride, in bytes
      constexpr bool kFixed = ALIGNED;
      const int lin = wave * 64 + lane;
      // (granule i lies kStep rows behind granule 0, where the swap is the same, or one of two in turn)
      constexpr int kStep = kThreads / kPRow, kTurns = kStep % 16 == 0 ? 1 : 2;
      static_assert(kStep % 8 == 0, "the swaps repeat");
      const char* zero = reinterpret_cast<const char*>(kZeroGranule);
      const char *dy0[kTurns], *x0[kTurns];
      unsigned dy_ld[kTurns], x_ld[kTurns];
#pragma unroll
      for (int h = 0; h < kTurns; ++h) {
        const int k = lin / kPRow + h * kStep;
        const int cd = m0 + ((lin % kPRow) ^ across_swap_p<T, BM>(k)) * kV;
        const int cx = n0 + ((lin % kPRow) ^ across_swap_q<T, BN>(k)) * kV;
        dy0[h] = cd < a.out ? reinterpret_cast<const char*>(static_cast<const T*>(a.dy) + cd) : zero;
        x0[h] = cx < a.k ? reinterpret_cast<const char*>(static_cast<const T*>(a.x) + cx) : zero;
        dy_ld[h] = cd < a.out ? (unsigned)(a.ld_dy * (int64_t)sizeof(T)) : 0u;
        x_ld[h] = cx < a.k ? (unsigned)(a.ld_x * (int64_t)sizeof(T)) : 0u;
      }
      // The workgroups of an XCD work on tiles of the same rows, each beginning its run somewhere in the
      // line.  Taking a tile's stages not from its first but from the one that a clock common to
      // all (units since the start, `done`) points at keeps them at the same rows at the same time,
      // and the rows in the L2 (65 536 rows, 16 groups of 2048 x 2048 bf16: 1.93 -> 1.46 GB fetched,
      // 823 -> 737 us).
      const int64_t turn = (done + stages - pl.stage % stages) % stages;
      auto place_of = [&](int64_t st) {
        const int64_t t = st + turn;
        return t < stages ? t : t - stages;
      };
      auto look = [&](int64_t st) {
        if (!a.order || wave != 0 || st >= stages) return;
        int64_t pos = r0 + place_of(st) * kK + (lane < kK ? lane : kK - 1);
        if (pos >= a.g.n) pos = a.g.n - 1;
        lds_load4(a.order + pos, reinterpret_cast<char*>(ids + (st & 1) * 64));
      };
      // load i: dy's and x's granules of one row
      constexpr int kLoads = kPLoads;
      u32x4 held[ALIGNED ? 1 : 2 * kLoads];
      const bool inside = m0 + BM <= a.out && n0 + BN <= a.k;
      // (through registers: each lane fetches its rows' numbers itself, a stage ahead)
      int rid[ALIGNED ? 1 : kLoads];
      auto row_of = [&](int i, int64_t st) {
        const int64_t pos = r0 + place_of(st) * kK + ((i * kWaves + wave) * 64 + lane) / kPRow;
        if (st >= stages || pos >= r1) return -1;
        return a.order ? a.order[pos] : (int)pos;
      };
      auto load = [&](int i, int64_t st, char* buf) {
        const int q0 = (i * kWaves + wave) * 64;
        const int64_t first = r0 + place_of(st) * kK;
        if (kFixed && first + kK <= r1) {
          // (behind the matrix a lane's pointer is that of the zeros, its row stride 0)
          const int k = lin / kPRow + i * kStep, h = i % kTurns;
          unsigned r = (unsigned)first + (unsigned)k;
          if (a.order) r = (unsigned)ids[(st & 1) * 64 + k];
          const bool in = r < (unsigned)a.g.n;
          const char* d = dy0[h] + (uint64_t)r * dy_ld[h];
          const char* x = x0[h] + (uint64_t)r * x_ld[h];
          lds_load16(in ? d : reinterpret_cast<const char*>(kZeroGranule), buf + q0 * 16);
          lds_load16(in ? x : reinterpret_cast<const char*>(kZeroGranule), buf + kPBytes + q0 * 16);
          return;
        }
        int q = q0 + lane;
        asm volatile("" : "+v"(q));   // (worked out at each load: there are no registers to keep it in)
        const int k = q / kPRow, s = q % kPRow;
        int r = (int)first + k;
        if constexpr (!ALIGNED) r = rid[i];
        else if (a.order) r = ids[(st & 1) * 64 + k];
        const bool in = k < r1 - first && (unsigned)r < (unsigned)a.g.n;
        const int cd = m0 + (s ^ across_swap_p<T, BM>(k)) * kV, cx = n0 + (s ^ across_swap_q<T, BN>(k)) * kV;
        const T* rd = static_cast<const T*>(a.dy) + (int64_t)r * a.ld_dy;
        const T* rx = static_cast<const T*>(a.x) + (int64_t)r * a.ld_x;
        if constexpr (ALIGNED) {
          fetch<T>(in ? rd : nullptr, cd, a.out, buf + q0 * 16);
          fetch<T>(in ? rx : nullptr, cx, a.k, buf + kPBytes + q0 * 16);
        } else if (inside) {
          __builtin_memcpy(&held[2 * i], in ? reinterpret_cast<const char*>(rd + cd) : zero, 16);
          __builtin_memcpy(&held[2 * i + 1], in ? reinterpret_cast<const char*>(rx + cx) : zero, 16);
        } else {
          held[2 * i] = granule_of<T>(in ? rd : nullptr, cd, a.out);
          held[2 * i + 1] = granule_of<T>(in ? rx : nullptr, cx, a.k);
        }
      };
      auto place = [&](int i, char* buf) {
        if constexpr (!ALIGNED) {
          const int at = ((i * kWaves + wave) * 64 + lane) * 16;
          *reinterpret_cast<u32x4*>(buf + at) = held[2 * i];
          *reinterpret_cast<u32x4*>(buf + kPBytes + at) = held[2 * i + 1];
        }
      };
      constexpr int kHalves = FM >= 4 ? 2 : 1, kHalf = FM / kHalves;
      u32x4 pf[2][kHalf], qf[2][FN];
      auto read_p = [&](const char* buf, int step, int half, int to) {
        read_fragments<T, BM, false, false, kHalf>(buf, pplace, step, half * kHalf, pf[to]);
      };
      auto read_q = [&](const char* buf, int step, int to) {
        read_fragments<T, BN, false, true, FN>(buf, qplace, step, 0, qf[to]);
      };
      // `count` loads are issued between the products
      auto mul = [&](int q, int half, int p, int count, auto&& issue) {
#pragma unroll
        for (int i = 0; i < kHalf; ++i) {
#pragma unroll
          for (int part = 0; part < Mma<T>::kParts; ++part)
#pragma unroll
            for (int j = 0; j < FN; ++j)
              acc[half * kHalf + i][j] = Mma<T>::mul(part, qf[q][j], pf[p][i], acc[half * kHalf + i][j]);
          if (count > 0) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int l = 0; l < kLoads; ++l)
              if (l < count && l * kHalf / count == i) issue(l);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      if constexpr (ALIGNED) {
        MULTIPLY_STAGES(stages, load, look, true, 2)
      } else {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) rid[i] = row_of(i, 0);
        auto fill = [&](int i, int64_t st) {
          load(i, st, smem);
          rid[i] = row_of(i, st + 1);
        };
        MULTIPLY_HELD(stages, fill, place)
      }
      __syncthreads();   // the buffers are free for the next run's loads
    }
    done += run;
    // (a.whole: always, unless the offsets do not ascend; there is no scratch then)
    const bool whole = a.whole || (pl.stage == 0 && run == pl.stages);
    if (whole) {
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        const int o = m0 + pc + i * 16 + (lane & 15);
        if (o < a.out) store16<T>(a.dw, (pl.e * a.out + o) * a.k, n0 + qc, a.k, lane, a.y_f32, acc[i]);
      }
    } else {
      // 16 bytes a lane, lanes side by side; the join undoes the order
      f32x4* part = reinterpret_cast<f32x4*>(a.part) +
                    (size_t)(2 * w + (pl.stage == 0 ? 1 : 0)) * (BM * BN / 4) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j) part[(i * FN + j) * kThreads] = acc[i][j];
    }
    if (u >= u1 || !dw_next(a, pl, kK)) break;
  }
}

// Adds the pieces of the tiles that are cut.  Workgroup row y stands for the end of run y of the line:
// if it lies inside a tile, the rows y of all the ends inside that tile share its elements, 64 f32x4 at a
// time, so that a tile cut into many pieces has as many workgroups to read them (100 000 rows, 1 group
// of 100 x 128 float32, 256 pieces a tile: 22 us, 467 with one).  Few pieces: each wave adds all
// of its 64, in the order of the line.  Many: the four waves share the pieces of the same 64, every
// fourth each, and their sums are added in the waves' order.  Either way the order depends on the sizes
// alone.
constexpr int kJoinWaves = 4;
constexpr int kJoinFew = 8;
template <typename T, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(kJoinWaves * 64) void k_grouped_dw_join(DwArgs a) {
  constexpr int kThreads = WM * WN * 64, kK = Mma<T>::kK, FN = 4;
  __shared__ f32x4 sums[kJoinWaves][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t w = blockIdx.y;
  const int64_t line = dw_line(a, kK);
  const int64_t u1 = line * (w + 1) / a.wgs;
  if (u1 >= line) return;
  const DwPlace pl = dw_place(a, u1, kK, lane);
  const int64_t begin = u1 - pl.stage, end = begin + pl.stages;
  if (pl.stage == 0 || begin < 0 || end > line) return;   // (outside only if the offsets do not ascend)
  // the workgroups that hold the tile's first and last unit; the ends of all but the last lie inside
  const int64_t first = ((begin + 1) * a.wgs - 1) / line, last = (end * a.wgs - 1) / line;
  constexpr int kTile = BM * BN / 4;
  const f32x4* part = reinterpret_cast<const f32x4*>(a.part);
  // workgroup v's piece of the tile; an empty run holds none
  auto piece = [&](int64_t v, int at) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    if (v == first) s = part[(size_t)(2 * v + 1) * kTile + at];
    else if (line * v / a.wgs != line * (v + 1) / a.wgs) s = part[(size_t)(2 * v) * kTile + at];
    return s;
  };
  auto put = [&](int at, f32x4 s) {
    // the lane of k_grouped_dw that wrote this f32x4, and which of its products
    const int t = at % kThreads, ij = at / kThreads;
    const int tl = t & 63, tw = t >> 6;
    const int o = pl.tile / a.k_tiles * BM + tw % WM * (BM / WM) + ij / FN * 16 + (tl & 15);
    const int c = pl.tile % a.k_tiles * BN + tw / WM * (BN / WN) + spread_row<T>((tl >> 4) * 4) +
                  spread_step<T>(ij % FN);
    if (o >= a.out) return;
    const int64_t to = (pl.e * a.out + o) * a.k + c;
    const int left = a.k - c;
    if (a.y_f32 || sizeof(T) == 4) {
      float* d = static_cast<float*>(a.dw) + to;
      if (left >= 4) {
        __builtin_memcpy(d, &s, 16);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < left) d[q] = s[q];
      }
    } else if constexpr (sizeof(T) == 2) {
      T* d = static_cast<T*>(a.dw) + to;
      if (left >= 4) {
        const float f[8] = {s[0], s[1], s[2], s[3], 0.f, 0.f, 0.f, 0.f};
        const u32x4 w = Elem<T>::pack(f);
        const u32x2 h = {w[0], w[1]};
        __builtin_memcpy(d, &h, 8);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < left) Elem<T>::store(d + q, s[q]);
      }
    }
  };
  const int mine = (int)((w - first) * gridDim.x + blockIdx.x);      // of this tile's workgroups
  const int all = (int)((last - first) * gridDim.x);
  if (last - first < kJoinFew) {
    for (int at = (mine * kJoinWaves + wave) * 64 + lane; at < kTile; at += all * kJoinWaves * 64) {
      f32x4 s = piece(first, at);
      for (int64_t v = first + 1; v <= last; ++v) s += piece(v, at);
      put(at, s);
    }
    return;
  }
  for (int at = mine * 64 + lane; at < kTile; at += all * 64) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    int64_t v = first + wave;
    for (; v + 7 * kJoinWaves <= last; v += 8 * kJoinWaves) {
      f32x4 q[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = piece(v + i * kJoinWaves, at);
#pragma unroll
      for (int i = 0; i < 8; ++i) s += q[i];
    }
    for (; v <= last; v += kJoinWaves) s += piece(v, at);
    sums[wave][lane] = s;
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int q = 1; q < kJoinWaves; ++q) s += sums[q][lane];
      put(at, s);
    }
    __syncthreads();
  }
}

template <int BM, int BN>
constexpr int rows_lds() { return 2 * (BM + BN) * kStageBytes + (BM > 128 ? BM : 128) * 4; }

// `tiles` workgroups, in more than one launch where their threads pass 32 bits.
template <typename Kernel>
hipError_t launch_tiles(Kernel kernel, RowsArgs a, int64_t tiles, int threads, int lds, hipStream_t s) {
  const int64_t most = 0xffffffffll / threads;
  for (a.id0 = 0; a.id0 < tiles; a.id0 += most) {
    const int64_t now = tiles - a.id0 < most ? tiles - a.id0 : most;
    hipLaunchKernelGGL(kernel, dim3((unsigned)now), dim3(threads), lds, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int BM, int BN, int WM, int WN, bool QALONG, bool ALIGNED>
hipError_t rows_launch(RowsArgs a, hipStream_t s) {
  a.col_tiles = (a.cols + BN - 1) / BN;
  return launch_tiles(k_grouped_rows<T, BM, BN, WM, WN, QALONG, ALIGNED>, a,
                      (a.g.n / BM + a.g.groups + 1) * a.col_tiles, WM * WN * 64, rows_lds<BM, BN>(), s);
}

// The tile sizes: workgroups of 256 x 256 (8 waves of 128 x 64, one workgroup a CU), 128 x 128 (4 waves
// of 64 x 64, two a CU) and 64 x 64 (4 waves of 16 x 64, four a CU).
constexpr int kTileSize[3] = {256, 128, 64};
constexpr int kPerCu[3] = {1, 2, 4};
// Rate of a full CU relative to 256 x 256 tiles (a smaller tile reads more of LDS and L2 a product;
// float32 products are eight to sixteen times slower and do not notice).  Measured with whole rounds of the card,
// TFLOP/s with tiles of 256, 128 and 64: bf16 forward 976, 748, 477, dw 1003, 660, 371; float32 forward
// 123, 122, 121, dw 124, 112, 100 (in dw both operands are read 4 bytes a lane, and a small tile reads more of
// them).  256 x 256 of float32 are held back because a group's last tile wastes more (16 groups of 1024 x 1024,
// forward: 108, 117, 118).
constexpr double kRate16[3] = {1.0, 0.8, 0.5}, kRate32[3] = {0.7, 1.0, 0.85};

// The tile with the least time for `tiles(size)` tiles: the most tiles that a CU gets times a tile's work, over
// the rate of as many workgroups as run there at a time (counting whole rounds of the card instead, 8192 rows,
// 16 groups of 2048 x 512 float32, dx, took 128 x 128 tiles: 275 us, with 64 x 64 199).
template <typename F>
int pick_tile(int type, bool aligned, F tiles) {
  // (not kRate32: 64 x 64 tiles of float32 lose 1 to 3 % of the rate of 128 x 128 here, 11 % in dw)
  static const double kRows32[3] = {0.7, 1.0, 0.97};
  const double* rate = type == IC_F32 ? kRows32 : kRate16;
  int best = 2;
  double least = 1e300;
  for (int i = aligned ? 0 : 1; i < 3; ++i) {
    const int64_t most = (tiles(kTileSize[i]) + kCUs - 1) / kCUs;
    const double busy = most < kPerCu[i] ? 0.2 + 0.8 * (double)most / kPerCu[i] : 1.0;
    const double t = (double)most * kTileSize[i] * kTileSize[i] / (rate[i] * busy);
    if (t < least) {
      least = t;
      best = i;
    }
  }
  return best;
}

template <typename T, int NS, bool QALONG>
hipError_t short_launch(RowsArgs a, hipStream_t s) {
  a.col_tiles = (a.cols + 63) / 64;
  // 128 rows a workgroup where there are many of them: the matrix is fetched and read from LDS for twice the
  // rows (1M rows, 2000 groups of 64 x 128 float32: 261 -> 246 us, 200 000 rows, 2000 groups of 200 x 64
  // bf16 45 -> 40); with few (20 000 rows, 200 groups: 11.4 -> 16.5) or narrow results (32 columns: 70 -> 74) 64
  const int64_t twice = (a.g.n / 128 + a.g.groups + 1) * a.col_tiles;
  if (twice >= 8192 && a.cols > 32) return launch_tiles(k_grouped_short<T, NS, 2, QALONG>, a, twice, 256, 0, s);
  return launch_tiles(k_grouped_short<T, NS, 1, QALONG>, a, (a.g.n / 64 + a.g.groups + 1) * a.col_tiles, 256, 0, s);
}

// Few rows.
template <typename T, bool QALONG, bool ALIGNED>
hipError_t few_launch(RowsArgs a, hipStream_t s) {
  const bool by_depth = !QALONG || a.depth >= 512;
  a.col_tiles = by_depth ? (a.cols + 31) / 32 : (a.cols + 63) / 64;
  const int64_t tiles = (a.g.n / 16 + a.g.groups + 1) * a.col_tiles;
  if (by_depth) return launch_tiles(k_grouped_few<T, true, QALONG, ALIGNED>, a, tiles, 256, 0, s);
  if constexpr (QALONG) return launch_tiles(k_grouped_few<T, false, true, ALIGNED>, a, tiles, 256, 0, s);
  return hipErrorInvalidValue;
}

template <typename T, bool QALONG>
hipError_t rows_typed(const RowsArgs& a, int type, bool aligned, hipStream_t s) {
  // rows in tiles of 16, without stages: few rows a group or in all; and where the depth is long and tiles
  // would leave most of the card idle (128 rows, 1 group of 1024 x 1024 float32: 28.5 -> 10.4 us, 250 rows,
  // 3 groups of 1001 -> 100 38 -> 9.4; but 256 rows, 4 groups of 2048 x 2048 bf16, 256 tiles: 24 -> 30)
  const int64_t tiles64 = (a.g.n / 64 + a.g.groups) * ((a.cols + 63) / 64);
  const bool idle = a.g.n <= 256 && tiles64 < 128;
  // (dx: 16-bit columns gathered element by element take longer than the stages do: 16 rows, 4 groups of
  // 2000 x 128 fp16 16.6 -> 29 us; float32 from a depth of 256 on: 2 rows, 410 -> 943, 19.7 -> 8.5 us)
  if constexpr (!QALONG && sizeof(T) == 4)
    if (idle && a.depth >= 256) return few_launch<T, false, false>(a, s);
  if constexpr (QALONG)
    if (a.g.n <= 8 * a.g.groups || a.g.n <= 32 || (idle && a.depth >= 512))
      return aligned ? few_launch<T, true, true>(a, s) : few_launch<T, true, false>(a, s);
  // rows of at most 512 bytes whose tiles would be 64 x 64 anyway (fewer columns, or short groups)
  const int64_t row_bytes = (int64_t)a.depth * (int)sizeof(T);
  if (aligned && row_bytes <= 512 && (a.cols <= 64 || a.g.n < 128 * a.g.groups)) {
    if (row_bytes <= 128) return short_launch<T, 1, QALONG>(a, s);
    if (row_bytes <= 256) return short_launch<T, 2, QALONG>(a, s);
    return short_launch<T, 4, QALONG>(a, s);
  }
  const int tile = pick_tile(type, aligned, [&](int size) {
    return (a.g.n / size + a.g.groups) * ((a.cols + size - 1) / size);
  });
  if (!aligned)
    return tile == 1 ? rows_launch<T, 128, 128, 2, 2, QALONG, false>(a, s)
                     : rows_launch<T, 64, 64, 4, 1, QALONG, false>(a, s);
  if (tile == 0) return rows_launch<T, 256, 256, 2, 4, QALONG, true>(a, s);
  if (tile == 1) return rows_launch<T, 128, 128, 2, 2, QALONG, true>(a, s);
  return rows_launch<T, 64, 64, 4, 1, QALONG, true>(a, s);
}

// Whether 16-byte granules can be loaded, and a row's stride in bytes fits 32 bits.
bool grouped_aligned(const GroupedCall& c, bool dw) {
  const int v = c.type == IC_F32 ? 4 : 8;
  const int b = c.type == IC_F32 ? 4 : 2;
  auto fits = [&](const void* p, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * b) % 16 == 0 && ld * b <= 0xffffffffll;
  };
  if (dw) return fits(c.x, c.ld_x) && fits(c.w, c.ld_w) && c.k % v == 0 && c.out % v == 0;
  return fits(c.x, c.ld_x) && fits(c.w, c.k) && c.k % v == 0 && c.out % v == 0;
}

// How dw runs: the tile with the least time for its part of the line, and how many workgroups.
struct DwPlan {
  int tile;
  int wgs;
  bool whole;
};
DwPlan dw_plan(int64_t n, int64_t groups, int k, int out, int type, bool aligned) {
  const int kk = kStageBytes / (type == IC_F32 ? 4 : 2);
  const double* rate = type == IC_F32 ? kRate32 : kRate16;
  DwPlan best = {2, 1, false};
  double least = 1e300;
  // Whole tiles, nothing cut and nothing joined: where a tile has at most five stages (128 rows, 1 group of
  // 1024 x 1024 float32: 21 -> 10 us with the call), and up to 128 where there are half as many groups as stages, so that
  // few tiles are long (4000 rows, 300 groups of 16 x 136 fp16: 20.2 -> 10.4 us, 2000 rows, 20 groups of 64 x 64
  // bf16 15.0 -> 12.5; but 8000 rows, 20 groups: 15.7 -> 26.4, and 1000 rows, 1 group: 13.7 -> 15.8).
  const int64_t stages = n / kk;
  const bool whole = stages <= 4 || (groups >= 4 && stages <= 128 && stages <= (groups > 8 ? 2 * groups : 16));
  for (int i = aligned ? 0 : 1; i < 3; ++i) {
    const int size = kTileSize[i];
    const double tiles = (double)((out + size - 1) / size) * ((k + size - 1) / size);
    const double line = ((double)(n / kk) + groups) * tiles;
    // at least four units a workgroup (5003 rows, 37 groups of 317 x 193 fp16, join included: 32.0 us with
    // at least six, 28.9 with four, 31.9 with two); a piece costs its partial result and the start of a
    // pipeline, the time of about six units
    double wgs = line / 4;
    const double slots = (double)kCUs * kPerCu[i];
    if (whole) {
      const double all = tiles * groups, rounds = std::ceil(all / slots);
      const double t = rounds * kPerCu[i] * size * size / rate[i];
      if (t < least) {
        least = t;
        best = DwPlan{i, (int)(all < 8 * slots ? all : 8 * slots), whole};
      }
      continue;
    }
    wgs = wgs < 1 ? 1 : wgs > slots ? slots : wgs;
    const double t = (line / wgs + 6) * kPerCu[i] * size * size / rate[i];
    if (t < least) {
      least = t;
      best = DwPlan{i, (int)wgs, false};
    }
  }
  return best;
}
size_t dw_scratch_of(const DwPlan& p) {
  return p.whole ? 0 : (size_t)2 * p.wgs * kTileSize[p.tile] * kTileSize[p.tile] * 4;
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
hipError_t dw_launch(DwArgs a, hipStream_t s) {
  a.k_tiles = (a.k + BN - 1) / BN;
  const int64_t tiles = (int64_t)((a.out + BM - 1) / BM) * a.k_tiles;
  if (tiles > 0x7fffffff) return hipErrorInvalidValue;
  a.tiles = (int)tiles;
  hipLaunchKernelGGL((k_grouped_dw<T, BM, BN, WM, WN, ALIGNED>), dim3((unsigned)a.wgs), dim3(WM * WN * 64),
                     (rows_lds<BM, BN>()), s, a);
  if (a.wgs > 1 && !a.whole) {
    // a workgroup for each 4096 elements and each end of a run; four where that makes few (2000 rows,
    // 8 groups of 64 x 128 float32, both kernels: 14.8 -> 12.5 us; with many, most find nothing to add and
    // more of them cost time: 4096 rows, 16 groups of 512 x 512 bf16, 23.7 us with one, 27.1 with four)
    constexpr int kEach = BM * BN / 4096;
    const int each = kEach * a.wgs <= 256 ? 4 * kEach : kEach;
    hipLaunchKernelGGL((k_grouped_dw_join<T, BM, BN, WM, WN>), dim3(each, (unsigned)(a.wgs - 1)),
                       dim3(kJoinWaves * 64), 0, s, a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t dw_typed(const DwArgs& a, int tile, bool aligned, hipStream_t s) {
  if (!aligned)
    return tile == 1 ? dw_launch<T, 128, 128, 2, 2, false>(a, s) : dw_launch<T, 64, 64, 4, 1, false>(a, s);
  if (tile == 0) return dw_launch<T, 256, 256, 2, 4, true>(a, s);
  if (tile == 1) return dw_launch<T, 128, 128, 2, 2, true>(a, s);
  return dw_launch<T, 64, 64, 4, 1, true>(a, s);
}

template <typename Kernel>
hipError_t allow(Kernel kernel, int bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <typename T>
hipError_t allow_typed() {
  hipError_t e = allow(k_grouped_rows<T, 128, 128, 2, 2, true, true>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_rows<T, 128, 128, 2, 2, true, false>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_rows<T, 128, 128, 2, 2, false, false>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_dw<T, 128, 128, 2, 2, false>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_rows<T, 128, 128, 2, 2, false, true>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_dw<T, 128, 128, 2, 2, true>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_rows<T, 256, 256, 2, 4, true, true>, rows_lds<256, 256>());
  if (e == hipSuccess) e = allow(k_grouped_rows<T, 256, 256, 2, 4, false, true>, rows_lds<256, 256>());
  if (e == hipSuccess) e = allow(k_grouped_dw<T, 256, 256, 2, 4, true>, rows_lds<256, 256>());
  return e;
}

}  // namespace

hipError_t grouped_init() {
  hipError_t e = allow_typed<float>();
  if (e == hipSuccess) e = allow_typed<bf16_t>();
  if (e == hipSuccess) e = allow_typed<f16_t>();
  return e;
}

size_t group_rows_scratch(int64_t n, int64_t groups) {
  return n <= kSmallRows ? 0 : sort_plan(n, groups).bytes;
}

hipError_t launch_group_rows(const int32_t* codes, int64_t n, int64_t groups, int32_t* order,
                             int64_t* offsets, void* scratch, hipStream_t s) {
  const SortPlan p = sort_plan(n, groups);
  if (n <= kSmallRows) {
    const int passes = (p.bits + kSmallBits - 1) / kSmallBits, bits = (p.bits + passes - 1) / passes;
    if (n <= 256)
      hipLaunchKernelGGL(k_group_small<256>, dim3(1), dim3(256), 0, s, codes, (int)n, groups, passes, bits,
                         order, offsets);
    else
      hipLaunchKernelGGL(k_group_small<1024>, dim3(1), dim3(1024), 0, s, codes, (int)n, groups, passes, bits,
                         order, offsets);
    return hipGetLastError();
  }
  char* ws = static_cast<char*>(scratch);
  unsigned* tab = reinterpret_cast<unsigned*>(ws + p.o_tab);
  unsigned* total = reinterpret_cast<unsigned*>(ws + p.o_total);
  Pair* pairs[2] = {reinterpret_cast<Pair*>(ws + p.o_pairs0), reinterpret_cast<Pair*>(ws + p.o_pairs1)};
  int32_t* sorted = reinterpret_cast<int32_t*>(ws + p.o_codes);
  const Pair* in = nullptr;
  for (int i = 0; i < p.passes; ++i) {
    const int shift = i * p.digit_bits;
    const bool few = p.rows == 2048;
    hipLaunchKernelGGL(few ? k_sort_count<2048> : k_sort_count<4096>, dim3((unsigned)p.blocks), dim3(kSortThreads), 0,
                       s, codes, in, n, groups, shift, p.digit_bits, tab);
    hipLaunchKernelGGL(k_sort_scan, dim3(1u << p.digit_bits), dim3(256), 0, s, tab, p.blocks, total);
    Pair* out = i + 1 < p.passes ? pairs[i & 1] : nullptr;
    hipLaunchKernelGGL(few ? k_sort_scatter<2048> : k_sort_scatter<4096>, dim3((unsigned)p.blocks), dim3(kSortThreads),
                       0, s, codes, in, n, groups, shift, p.digit_bits, tab, total, out, order, sorted);
    in = out;
  }
  hipLaunchKernelGGL(k_group_offsets, dim3((unsigned)((n + 1 + 255) / 256)), dim3(256), 0, s, sorted, n, groups,
                     offsets);
  return hipGetLastError();
}

hipError_t launch_grouped_rows(const GroupedCall& c, bool dx, hipStream_t s) {
  RowsArgs a;
  a.p = c.x;
  a.q = c.w;
  a.y = c.y;
  a.g = Groups{c.offsets, c.n, c.groups};
  a.order = c.order;
  a.ld_p = c.ld_x;
  a.ld_q = c.k;
  a.ld_y = c.ld_y;
  a.q_stride = (int64_t)c.out * c.k;
  a.depth = dx ? c.out : c.k;
  a.cols = dx ? c.k : c.out;
  a.y_f32 = c.y_f32 || c.type == IC_F32;
  const bool al = grouped_aligned(c, false);
  if (c.type == IC_F32) return dx ? rows_typed<float, false>(a, c.type, al, s) : rows_typed<float, true>(a, c.type, al, s);
  if (c.type == IC_BF16) return dx ? rows_typed<bf16_t, false>(a, c.type, al, s) : rows_typed<bf16_t, true>(a, c.type, al, s);
  return dx ? rows_typed<f16_t, false>(a, c.type, al, s) : rows_typed<f16_t, true>(a, c.type, al, s);
}

size_t grouped_dw_scratch(int64_t n, int64_t groups, int k, int out, int type) {
  const size_t a = dw_scratch_of(dw_plan(n, groups, k, out, type, true));
  const size_t b = dw_scratch_of(dw_plan(n, groups, k, out, type, false));
  return a > b ? a : b;
}

hipError_t launch_grouped_dw(const GroupedCall& c, void* scratch, hipStream_t s) {
  const bool al = grouped_aligned(c, true);
  DwArgs a;
  a.dy = c.w;
  a.x = c.x;
  a.dw = c.y;
  a.part = static_cast<float*>(scratch);
  a.g = Groups{c.offsets, c.n, c.groups};
  a.order = c.order;
  a.ld_dy = c.ld_w;
  a.ld_x = c.ld_x;
  const DwPlan plan = dw_plan(c.n, c.groups, c.k, c.out, c.type, al);
  a.wgs = plan.wgs;
  a.whole = plan.whole;
  a.out = c.out;
  a.k = c.k;
  a.y_f32 = c.y_f32 || c.type == IC_F32;
  if (c.type == IC_F32) return dw_typed<float>(a, plan.tile, al, s);
  if (c.type == IC_BF16) return dw_typed<bf16_t>(a, plan.tile, al, s);
  return dw_typed<f16_t>(a, plan.tile, al, s);
}

}  // namespace ic
