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
#include "ic_wave.h"

namespace ic {

namespace {

static __device__ __align__(16) const unsigned kZeroGranule[4] = {0u, 0u, 0u, 0u};

// ---- group_rows ----------------------------------------------------------------------------------
constexpr int kSmallRows = 4096;

// Few rows: one workgroup sorts (group << 12 | row) in LDS.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_group_small(const int32_t* __restrict__ codes, int n,
                                                         int64_t groups, int32_t* __restrict__ order,
                                                         int64_t* __restrict__ offsets) {
  __shared__ unsigned buf[kSmallRows];
  int P = 2 * THREADS;
  while (P < n) P <<= 1;
  for (int p = threadIdx.x; p < P; p += THREADS) {
    unsigned key = 0xffffffffu;
    if (p < n) {
      const int32_t c = codes[p];
      const unsigned g = c >= 0 && c < groups ? (unsigned)c : 0xfffffu;
      key = (g << 12) | (unsigned)p;
    }
    buf[p] = key;
  }
  for (int size = 2; size <= P; size <<= 1) {
    for (int stride = size >> 1; stride > 0; stride >>= 1) {
      __syncthreads();
      for (int t = threadIdx.x; t < P / 2; t += THREADS) {
        const int pos = 2 * t - (t & (stride - 1));
        const unsigned a = buf[pos], b = buf[pos + stride];
        if ((a > b) == ((pos & size) == 0)) {
          buf[pos] = b;
          buf[pos + stride] = a;
        }
      }
    }
  }
  __syncthreads();
  for (int p = threadIdx.x; p < n; p += THREADS) order[p] = (int32_t)(buf[p] & 4095u);
  // (rows of no group carry the key 0xfffff, which is behind every group)
  for (int64_t e = threadIdx.x; e <= groups; e += THREADS) {
    const unsigned want = (e == groups ? 0xfffffu : (unsigned)e) << 12;
    int lo = 0, hi = n;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (buf[mid] < want) lo = mid + 1; else hi = mid;
    }
    offsets[e] = lo;
  }
}

// Many rows: a least-significant-digit radix sort of (group, row) pairs, digits of up to 9 bits.
constexpr int kSortRows = 4096;     // rows of a workgroup
constexpr int kSortThreads = 1024;
constexpr int kSortWaves = kSortThreads / 64;
constexpr int kMaxDigitBits = 9;

struct SortPlan {
  int bits;        // of the key: groups + 1 values, the last for rows of no group
  int passes;
  int digit_bits;
  int64_t blocks;
  size_t o_tab, o_total, o_pairs0, o_pairs1, o_codes, bytes;
};
SortPlan sort_plan(int64_t n, int64_t groups) {
  SortPlan p;
  p.bits = 1;
  while (((int64_t)1 << p.bits) < groups + 1) ++p.bits;
  p.passes = (p.bits + kMaxDigitBits - 1) / kMaxDigitBits;
  p.digit_bits = (p.bits + p.passes - 1) / p.passes;
  p.blocks = (n + kSortRows - 1) / kSortRows;
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
__global__ __launch_bounds__(kSortThreads) void k_sort_count(const int32_t* codes, const Pair* pairs,
                                                             int64_t n, int64_t groups, int shift,
                                                             int digit_bits, unsigned* tab) {
  __shared__ unsigned cnt[1 << kMaxDigitBits];
  const int digits = 1 << digit_bits;
  for (int d = threadIdx.x; d < digits; d += kSortThreads) cnt[d] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * kSortRows;
#pragma unroll
  for (int r = 0; r < kSortRows / kSortThreads; ++r) {
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
  constexpr int kR = kSortRows / kSortThreads;   // rounds of 64 rows a wave
  const int64_t base = (int64_t)blockIdx.x * kSortRows + wave * (64 * kR);
  unsigned key[kR], rank[kR];
  const unsigned long long below = (1ull << lane) - 1ull;
#pragma unroll
  for (int r = 0; r < kR; ++r) {
    const int64_t i = base + r * 64 + lane;
    const bool in = i < n;
    key[r] = in ? key_of(codes, pairs, i, groups) : 0u;
    const unsigned d = (key[r] >> shift) & (digits - 1);
    unsigned long long same = __ballot(in);
    for (int b = 0; b < digit_bits; ++b) {
      const unsigned long long ones = __ballot((d >> b) & 1u);
      same &= ((d >> b) & 1u) ? ones : ~ones;
    }
    // (only this wave touches its counters: lanes of equal digit read before the first one adds)
    const unsigned old = cnt[wave][d];
    rank[r] = old + __popcll(same & below);
    __builtin_amdgcn_wave_barrier();
    if (in && (same & below) == 0) cnt[wave][d] = old + __popcll(same);
    __builtin_amdgcn_wave_barrier();
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

// The last e in [0, groups] whose first tile, at(e) / bm + e, is <= tile.  Every lane of the wave
// takes part and gets the answer.
__device__ __forceinline__ int64_t find_group(const Groups& g, int64_t tile, int64_t bm, int lane) {
  int64_t lo = 0, hi = g.groups + 1;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) >> 6;
    const int64_t e = lo + lane * step;
    const bool yes = e < hi && g.at(e) / bm + e <= tile;
    int c = __popcll(__ballot(yes));
    c = c > 1 ? c - 1 : 0;
    lo += c * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  const unsigned low = __builtin_amdgcn_readfirstlane((unsigned)lo);
  const unsigned high = __builtin_amdgcn_readfirstlane((unsigned)((uint64_t)lo >> 32));
  return (int64_t)(((uint64_t)high << 32) | low);
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

__device__ __forceinline__ void lds_load16(const void* src, char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

template <typename T> struct Mma;
template <> struct Mma<float> {
  static constexpr int kK = kStageBytes / 4;
  // a granule of each operand: 4 products deep in k (the lane's granule, one element a product; the
  // order of k inside a step is the same for both operands and does not matter)
  static __device__ __forceinline__ f32x4 mul(u32x4 q, u32x4 p, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(q[j]), __uint_as_float(p[j]), c, 0, 0, 0);
    return c;
  }
};
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <> struct Mma<bf16_t> {
  static constexpr int kK = kStageBytes / 2;
  static __device__ __forceinline__ f32x4 mul(u32x4 q, u32x4 p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q),
                                                   __builtin_bit_cast(bf16x8, p), c, 0, 0, 0);
  }
};
template <> struct Mma<f16_t> {
  static constexpr int kK = kStageBytes / 2;
  static __device__ __forceinline__ f32x4 mul(u32x4 q, u32x4 p, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, q),
                                                  __builtin_bit_cast(f16x8, p), c, 0, 0, 0);
  }
};

// Tile "along": [rows][128 bytes], granule s of row r holds granule s ^ (r & 7) of the stage.
__device__ __forceinline__ u32x4 read_along(const char* tile, int r0, int step, int lane) {
  const int r = r0 + (lane & 15);
  const int s = (step * 4 + (lane >> 4)) ^ (r & 7);
  return *reinterpret_cast<const u32x4*>(tile + r * kStageBytes + s * 16);
}

// Tile "across": [kK rows of the contraction][COLS], granules exchanged by the contraction row.
template <typename T>
__device__ __forceinline__ int across_swap(int k) {
  return sizeof(T) == 2 ? (k & 3) << 1 : ((k >> 2) & 3) << 2;
}
template <typename T, int COLS>
__device__ __forceinline__ u32x4 read_across(const char* tile, int c0, int step, int lane) {
  constexpr int kRow = COLS * (int)sizeof(T);
  u32x4 out;
  if constexpr (sizeof(T) == 2) {
    // the 16 lanes of a quarter wave point at 4 rows of the contraction x 16 columns, 4 columns
    // each; lane i is handed column i of the 4 rows
    const int t = lane & 15;
    const int s = ((c0 >> 3) + ((t & 3) >> 1)) ^ across_swap<T>(t >> 2);
    const char* p = tile + (step * 32 + (lane >> 4) * 8 + (t >> 2)) * kRow + s * 16 + (t & 1) * 8;
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
    const int t = lane & 15;
    const int s = ((c0 >> 2) + (t >> 2)) ^ across_swap<T>((lane >> 4) * 4);
    const char* p = tile + (step * 16 + (lane >> 4) * 4) * kRow + s * 16 + (t & 3) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) out[j] = *reinterpret_cast<const unsigned*>(p + j * kRow);
  }
  return out;
}

// One granule of an operand: elements [c, c + kVec) of a row of `cols` elements (NULL row: zeros).
template <typename T, bool ALIGNED>
__device__ __forceinline__ void fetch(const T* row, int64_t c, int64_t cols, char* lds_wave_base, int lane) {
  constexpr int kV = Elem<T>::kVec;
  if constexpr (ALIGNED) {
    const void* src = row && c < cols ? static_cast<const void*>(row + c)
                                      : static_cast<const void*>(kZeroGranule);
    lds_load16(src, lds_wave_base);
  } else {
    u32x4 w = {0u, 0u, 0u, 0u};
    if (row) {
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
    *reinterpret_cast<u32x4*>(lds_wave_base + lane * 16) = w;
  }
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
  int y_f32, y_vec;    // y_vec: four columns can be stored at once
};

// four neighbouring results of one row
template <typename T>
__device__ __forceinline__ void store4(void* y, int64_t at, int left, bool f32, bool vec, f32x4 v) {
  if (left <= 0) return;
  if (f32 || sizeof(T) == 4) {
    float* d = static_cast<float*>(y) + at;
    if (vec && left >= 4) {
      *reinterpret_cast<f32x4*>(d) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) d[i] = v[i];
    }
  } else if constexpr (sizeof(T) == 2) {
    T* d = static_cast<T*>(y) + at;
    if (vec && left >= 4) {
      T h[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) Elem<T>::store(&h[i], v[i]);
      *reinterpret_cast<u32x2*>(d) = *reinterpret_cast<u32x2*>(h);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < left) Elem<T>::store(d + i, v[i]);
    }
  }
}

// forward (QALONG: W_g [cols][depth]) and dx (W_g [depth][cols])
template <typename T, int BM, int BN, int WM, int WN, bool QALONG, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_grouped_rows(RowsArgs a) {
  constexpr int kThreads = WM * WN * 64, kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int kV = Elem<T>::kVec, kK = Mma<T>::kK;
  constexpr int kPBytes = BM * kStageBytes, kQBytes = BN * kStageBytes;
  constexpr int kPLoads = BM * 8 / kThreads, kQLoads = BN * 8 / kThreads;
  constexpr int kQRow = BN * (int)sizeof(T) / 16;   // granules of a contraction row (across)
  static_assert(kPLoads * kThreads == BM * 8 && kQLoads * kThreads == BN * 8, "tile");
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  int* rows = reinterpret_cast<int*>(smem + 2 * (kPBytes + kQBytes));
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = xcd_run(blockIdx.x, gridDim.x);
  const int64_t tile = id / a.col_tiles;
  const int c0 = (int)(id % a.col_tiles) * BN;
  const int64_t e = find_group(a.g, tile, BM, lane);
  const int64_t o0 = a.g.at(e), o1 = a.g.at(e + 1);
  const int64_t t = tile - (o0 / BM + e);
  const int64_t r0 = o0 + t * BM;
  if (t < 0 || r0 >= o1) return;   // (t < 0: only if the offsets do not ascend)
  const int m = o1 - r0 < BM ? (int)(o1 - r0) : BM;
  // the rows' numbers; -1 behind the group's end and for an entry of `order` that is no row
  for (int i = threadIdx.x; i < BM; i += kThreads) {
    int64_t r = -1;
    if (i < m) {
      r = a.order ? (int64_t)a.order[r0 + i] : r0 + i;
      if (r < 0 || r >= a.g.n) r = -1;
    }
    rows[i] = (int)r;
  }
  __syncthreads();
  const int wm = wave % WM, wn = wave / WM;
  const int pr = wm * (BM / WM), qc = wn * (BN / WN);
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  if (e < a.g.groups) {
    const T* qb = static_cast<const T*>(a.q) + e * a.q_stride;
    // this lane's granules: the row and the first element inside the stage
    const T* prow[kPLoads];
    const T* qrow[kQLoads];
#pragma unroll
    for (int i = 0; i < kPLoads; ++i) {
      const int r = ((i * kWaves + wave) * 64 + lane) >> 3;
      const int row = rows[r];
      // (a tile's rows behind the group's end are multiplied too and not stored)
      prow[i] = row >= 0 ? static_cast<const T*>(a.p) + (int64_t)row * a.ld_p : nullptr;
    }
#pragma unroll
    for (int i = 0; i < kQLoads; ++i) {
      const int q = (i * kWaves + wave) * 64 + lane;
      if (QALONG) {
        const int c = c0 + (q >> 3);
        qrow[i] = c < a.cols ? qb + (int64_t)c * a.ld_q : nullptr;
      } else {
        qrow[i] = qb + (int64_t)(q / kQRow) * a.ld_q;
      }
    }
    auto issue = [&](int st, char* buf) {
      const int64_t k0 = (int64_t)st * kK;
#pragma unroll
      for (int i = 0; i < kPLoads; ++i) {
        const int q0 = (i * kWaves + wave) * 64, q = q0 + lane;
        fetch<T, ALIGNED>(prow[i], k0 + ((q & 7) ^ ((q >> 3) & 7)) * kV, a.depth, buf + q0 * 16, lane);
      }
#pragma unroll
      for (int i = 0; i < kQLoads; ++i) {
        const int q0 = (i * kWaves + wave) * 64, q = q0 + lane;
        char* to = buf + kPBytes + q0 * 16;
        if (QALONG) {
          fetch<T, ALIGNED>(qrow[i], k0 + ((q & 7) ^ ((q >> 3) & 7)) * kV, a.depth, to, lane);
        } else {
          const int k = q / kQRow;
          const int c = c0 + ((q % kQRow) ^ across_swap<T>(k)) * kV;
          fetch<T, ALIGNED>(k0 + k < a.depth ? qrow[i] + k0 * a.ld_q : nullptr, c, a.cols, to, lane);
        }
      }
    };
    const int stages = (int)(((int64_t)a.depth + kK - 1) / kK);
    issue(0, smem);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int st = 0; st < stages; ++st) {
      char* buf = smem + (st & 1) * (kPBytes + kQBytes);
      if (st + 1 < stages) issue(st + 1, smem + ((st + 1) & 1) * (kPBytes + kQBytes));
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        u32x4 pf[FM], qf[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) pf[i] = read_along(buf, pr + i * 16, step, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j)
          qf[j] = QALONG ? read_along(buf + kPBytes, qc + j * 16, step, lane)
                         : read_across<T, BN>(buf + kPBytes, qc + j * 16, step, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::mul(qf[j], pf[i], acc[i][j]);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
  }
  // lane: row pr + 16 i + (lane & 15), columns qc + 16 j + 4 (lane >> 4) ..
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int row = rows[pr + i * 16 + (lane & 15)];
    if (row < 0) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int c = c0 + qc + j * 16 + (lane >> 4) * 4;
      store4<T>(a.y, (int64_t)row * a.ld_y + c, a.cols - c, a.y_f32, a.y_vec, acc[i][j]);
    }
  }
}

// ---- dw ---------------------------------------------------------------------------------------------
// dW_e[o][k] = sum_r dy[r][o] x[r][k]: both operands run across the contraction.  A group's rows are
// cut into chunks of `chunk` rows (tile numbers as above); a group of one chunk is written at once, the
// chunks of a longer one go to float32 partial results, which k_grouped_dw_join adds in chunk order.
// Chunk t of group e has partial result number 2 floor(o_e / chunk) + t: groups of more than one
// chunk have more than `chunk` rows, so 2 floor(rows / chunk) >= ceil(rows / chunk) numbers lie
// between their first ones, and 2 floor(n / chunk) of them are enough.
struct DwArgs {
  const void* dy;
  const void* x;
  void* dw;
  float* part;
  Groups g;
  const int32_t* order;
  int64_t ld_dy, ld_x;
  int64_t chunk;
  int out, k;
  int out_tiles, k_tiles;
  int y_f32, y_vec;
};

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
__global__ __launch_bounds__(WM * WN * 64) void k_grouped_dw(DwArgs a) {
  constexpr int kThreads = WM * WN * 64, kWaves = WM * WN;
  constexpr int FM = BM / WM / 16, FN = BN / WN / 16;
  constexpr int kV = Elem<T>::kVec, kK = Mma<T>::kK;
  constexpr int kPBytes = BM * kStageBytes, kQBytes = BN * kStageBytes;
  constexpr int kPLoads = BM * 8 / kThreads, kQLoads = BN * 8 / kThreads;
  constexpr int kPRow = BM * (int)sizeof(T) / 16, kQRow = BN * (int)sizeof(T) / 16;
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t id = xcd_run(blockIdx.x, gridDim.x);
  const int tiles = a.out_tiles * a.k_tiles;
  const int64_t tile = id / tiles;
  const int in_tile = (int)(id % tiles);
  const int m0 = in_tile / a.k_tiles * BM, n0 = in_tile % a.k_tiles * BN;
  const int64_t e = find_group(a.g, tile, a.chunk, lane);
  if (e >= a.g.groups) return;
  const int64_t o0 = a.g.at(e), o1 = a.g.at(e + 1);
  const int64_t t = tile - (o0 / a.chunk + e);
  const int64_t r0 = o0 + t * a.chunk;
  if (t < 0 || (r0 >= o1 && t != 0)) return;   // (the first tile of an empty group writes its zeros)
  const int64_t r1 = r0 + a.chunk < o1 ? r0 + a.chunk : o1;
  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int wm = wave % WM, wn = wave / WM;
  const int pc = wm * (BM / WM), qc = wn * (BN / WN);
  if (r0 < r1) {
    // a position's row: -1 behind the chunk
    auto row_at = [&](int64_t pos) {
      if (pos >= r1) return -1;
      const int64_t r = a.order ? (int64_t)a.order[pos] : pos;
      return r >= 0 && r < a.g.n ? (int)r : -1;
    };
    int prow[kPLoads], qrow[kQLoads];
    auto look = [&](int st) {
      const int64_t k0 = r0 + (int64_t)st * kK;
#pragma unroll
      for (int i = 0; i < kPLoads; ++i) prow[i] = row_at(k0 + ((i * kWaves + wave) * 64 + lane) / kPRow);
#pragma unroll
      for (int i = 0; i < kQLoads; ++i) qrow[i] = row_at(k0 + ((i * kWaves + wave) * 64 + lane) / kQRow);
    };
    auto issue = [&](char* buf) {
#pragma unroll
      for (int i = 0; i < kPLoads; ++i) {
        const int q0 = (i * kWaves + wave) * 64, q = q0 + lane;
        const int c = m0 + ((q % kPRow) ^ across_swap<T>(q / kPRow)) * kV;
        const T* row = prow[i] >= 0 ? static_cast<const T*>(a.dy) + (int64_t)prow[i] * a.ld_dy : nullptr;
        fetch<T, ALIGNED>(row, c, a.out, buf + q0 * 16, lane);
      }
#pragma unroll
      for (int i = 0; i < kQLoads; ++i) {
        const int q0 = (i * kWaves + wave) * 64, q = q0 + lane;
        const int c = n0 + ((q % kQRow) ^ across_swap<T>(q / kQRow)) * kV;
        const T* row = qrow[i] >= 0 ? static_cast<const T*>(a.x) + (int64_t)qrow[i] * a.ld_x : nullptr;
        fetch<T, ALIGNED>(row, c, a.k, buf + kPBytes + q0 * 16, lane);
      }
    };
    const int stages = (int)((r1 - r0 + kK - 1) / kK);
    look(0);
    issue(smem);
    look(1);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    for (int st = 0; st < stages; ++st) {
      char* buf = smem + (st & 1) * (kPBytes + kQBytes);
      if (st + 1 < stages) {
        issue(smem + ((st + 1) & 1) * (kPBytes + kQBytes));
        look(st + 2);
      }
#pragma unroll
      for (int step = 0; step < 2; ++step) {
        u32x4 pf[FM], qf[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) pf[i] = read_across<T, BM>(buf, pc + i * 16, step, lane);
#pragma unroll
        for (int j = 0; j < FN; ++j) qf[j] = read_across<T, BN>(buf + kPBytes, qc + j * 16, step, lane);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = Mma<T>::mul(qf[j], pf[i], acc[i][j]);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
    }
  }
  const bool whole = o1 - o0 <= a.chunk;
  const int64_t slot = whole ? e : 2 * (o0 / a.chunk) + t;
  void* to = whole ? a.dw : static_cast<void*>(a.part);
  const bool f32 = !whole || a.y_f32;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    const int o = m0 + pc + i * 16 + (lane & 15);
    if (o >= a.out) continue;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int c = n0 + qc + j * 16 + (lane >> 4) * 4;
      store4<T>(to, (slot * a.out + o) * a.k + c, a.k - c, f32, a.y_vec, acc[i][j]);
    }
  }
}

// Adds the chunks of the groups of more than one.  Such a group has more than `chunk` rows and holds
// exactly one position j * chunk in [o_e, o_e + chunk): workgroup row j looks for it.
template <typename T>
__global__ __launch_bounds__(256) void k_grouped_dw_join(DwArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t pos = (int64_t)blockIdx.y * a.chunk;
  if (pos >= a.g.n) return;
  // the group that holds position pos: the last e with at(e) <= pos (empty groups pushed aside)
  int64_t lo = 0, hi = a.g.groups + 1;
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) >> 6;
    const int64_t e = lo + lane * step;
    int c = __popcll(__ballot(e < hi && a.g.at(e) <= pos));
    c = c > 1 ? c - 1 : 0;
    lo += c * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  if (lo >= a.g.groups) return;
  const int64_t o0 = a.g.at(lo), rows = a.g.at(lo + 1) - o0;
  if (rows <= a.chunk || (o0 + a.chunk - 1) / a.chunk != (int64_t)blockIdx.y) return;
  const int64_t chunks = (rows + a.chunk - 1) / a.chunk;
  const int64_t size = (int64_t)a.out * a.k;
  const float* part = a.part + 2 * (o0 / a.chunk) * size;
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (int64_t)gridDim.x * 1024) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    const int left = size - i < 4 ? (int)(size - i) : 4;
    for (int64_t t = 0; t < chunks; ++t) {
      if (a.y_vec) {
        s += *reinterpret_cast<const f32x4*>(part + t * size + i);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (q < left) s[q] += part[t * size + i + q];
      }
    }
    store4<T>(a.dw, lo * size + i, left, a.y_f32, a.y_vec, s);
  }
}

template <int BM, int BN>
constexpr int rows_lds() { return 2 * (BM + BN) * kStageBytes + BM * 4; }

template <typename T, int BM, int BN, int WM, int WN, bool QALONG, bool ALIGNED>
hipError_t rows_launch(RowsArgs a, hipStream_t s) {
  a.col_tiles = (a.cols + BN - 1) / BN;
  const int64_t grid = (a.g.n / BM + a.g.groups + 1) * a.col_tiles;
  if (grid * (WM * WN * 64) > 0xffffffffll) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_grouped_rows<T, BM, BN, WM, WN, QALONG, ALIGNED>), dim3((unsigned)grid),
                     dim3(WM * WN * 64), (rows_lds<BM, BN>()), s, a);
  return hipGetLastError();
}

template <typename T, bool QALONG>
hipError_t rows_typed(const RowsArgs& a, bool aligned, hipStream_t s) {
  if (!aligned) return rows_launch<T, 64, 64, 2, 2, QALONG, false>(a, s);
  return rows_launch<T, 128, 128, 2, 2, QALONG, true>(a, s);
}

// Rows of a chunk: 2048 workgroups where the groups are long, at least 512 rows, and partial
// results of at most 256 MB.
int64_t dw_chunk(int64_t n, int out, int k) {
  const int64_t tiles = (int64_t)((out + 127) / 128) * ((k + 127) / 128);
  int64_t chunk = (n * tiles + 2047) / 2048;
  const int64_t bytes = 2 * n * (int64_t)out * k * 4;
  const int64_t by_memory = (bytes + ((int64_t)1 << 28) - 1) >> 28;
  if (chunk < by_memory) chunk = by_memory;
  if (chunk < 512) chunk = 512;
  return (chunk + 63) / 64 * 64;
}

bool grouped_aligned(const GroupedCall& c, bool dw) {
  const int v = c.type == IC_F32 ? 4 : 8;
  const int b = c.type == IC_F32 ? 4 : 2;
  auto fits = [&](const void* p, int64_t ld) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * b) % 16 == 0;
  };
  if (dw) return fits(c.x, c.ld_x) && fits(c.w, c.ld_w) && c.k % v == 0 && c.out % v == 0;
  return fits(c.x, c.ld_x) && fits(c.w, c.k) && c.k % v == 0 && c.out % v == 0;
}

template <typename T, int BM, int BN, int WM, int WN, bool ALIGNED>
hipError_t dw_launch(DwArgs a, hipStream_t s) {
  a.out_tiles = (a.out + BM - 1) / BM;
  a.k_tiles = (a.k + BN - 1) / BN;
  const int64_t grid = (a.g.n / a.chunk + a.g.groups + 1) * a.out_tiles * a.k_tiles;
  if (grid * (WM * WN * 64) > 0xffffffffll) return hipErrorInvalidValue;
  hipLaunchKernelGGL((k_grouped_dw<T, BM, BN, WM, WN, ALIGNED>), dim3((unsigned)grid), dim3(WM * WN * 64),
                     (rows_lds<BM, BN>()), s, a);
  if (a.g.n > a.chunk) {
    int64_t x = ((int64_t)a.out * a.k + 1023) / 1024;
    if (x > 4096) x = 4096;
    const int64_t y = (a.g.n + a.chunk - 1) / a.chunk;
    if (y > 65535) return hipErrorInvalidValue;
    hipLaunchKernelGGL(k_grouped_dw_join<T>, dim3((unsigned)x, (unsigned)y), dim3(256), 0, s, a);
  }
  return hipGetLastError();
}

template <typename T>
hipError_t dw_typed(DwArgs a, bool aligned, hipStream_t s) {
  if (!aligned) return dw_launch<T, 64, 64, 2, 2, false>(a, s);
  return dw_launch<T, 128, 128, 2, 2, true>(a, s);
}

template <typename Kernel>
hipError_t allow(Kernel kernel, int bytes) {
  return hipFuncSetAttribute(reinterpret_cast<const void*>(kernel),
                             hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}
template <typename T>
hipError_t allow_typed() {
  hipError_t e = allow(k_grouped_rows<T, 128, 128, 2, 2, true, true>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_rows<T, 128, 128, 2, 2, false, true>, rows_lds<128, 128>());
  if (e == hipSuccess) e = allow(k_grouped_dw<T, 128, 128, 2, 2, true>, rows_lds<128, 128>());
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
  if (n <= kSmallRows && groups <= 0xfffff) return 0;
  return sort_plan(n, groups).bytes;
}

hipError_t launch_group_rows(const int32_t* codes, int64_t n, int64_t groups, int32_t* order,
                             int64_t* offsets, void* scratch, hipStream_t s) {
  if (n <= kSmallRows && groups <= 0xfffff) {
    if (n <= 512)
      hipLaunchKernelGGL(k_group_small<256>, dim3(1), dim3(256), 0, s, codes, (int)n, groups, order, offsets);
    else
      hipLaunchKernelGGL(k_group_small<1024>, dim3(1), dim3(1024), 0, s, codes, (int)n, groups, order, offsets);
    return hipGetLastError();
  }
  const SortPlan p = sort_plan(n, groups);
  char* ws = static_cast<char*>(scratch);
  unsigned* tab = reinterpret_cast<unsigned*>(ws + p.o_tab);
  unsigned* total = reinterpret_cast<unsigned*>(ws + p.o_total);
  Pair* pairs[2] = {reinterpret_cast<Pair*>(ws + p.o_pairs0), reinterpret_cast<Pair*>(ws + p.o_pairs1)};
  int32_t* sorted = reinterpret_cast<int32_t*>(ws + p.o_codes);
  const Pair* in = nullptr;
  for (int i = 0; i < p.passes; ++i) {
    const int shift = i * p.digit_bits;
    hipLaunchKernelGGL(k_sort_count, dim3((unsigned)p.blocks), dim3(kSortThreads), 0, s, codes, in, n, groups,
                       shift, p.digit_bits, tab);
    hipLaunchKernelGGL(k_sort_scan, dim3(1u << p.digit_bits), dim3(256), 0, s, tab, p.blocks, total);
    Pair* out = i + 1 < p.passes ? pairs[i & 1] : nullptr;
    hipLaunchKernelGGL(k_sort_scatter, dim3((unsigned)p.blocks), dim3(kSortThreads), 0, s, codes, in, n,
                       groups, shift, p.digit_bits, tab, total, out, order, sorted);
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
  const int yb = a.y_f32 ? 4 : 2;
  a.y_vec = (reinterpret_cast<uintptr_t>(c.y) % (4 * yb)) == 0 && c.ld_y % 4 == 0;
  const bool al = grouped_aligned(c, false);
  if (c.type == IC_F32) return dx ? rows_typed<float, false>(a, al, s) : rows_typed<float, true>(a, al, s);
  if (c.type == IC_BF16) return dx ? rows_typed<bf16_t, false>(a, al, s) : rows_typed<bf16_t, true>(a, al, s);
  return dx ? rows_typed<f16_t, false>(a, al, s) : rows_typed<f16_t, true>(a, al, s);
}

size_t grouped_dw_scratch(int64_t n, int out, int k) {
  const int64_t chunk = dw_chunk(n, out, k);
  return n <= chunk ? 0 : (size_t)(2 * (n / chunk)) * out * k * 4;
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
  a.chunk = dw_chunk(c.n, c.out, c.k);
  a.out = c.out;
  a.k = c.k;
  a.y_f32 = c.y_f32 || c.type == IC_F32;
  a.y_vec = (reinterpret_cast<uintptr_t>(c.y) & 15) == 0 && c.k % 4 == 0;
  if (c.type == IC_F32) return dw_typed<float>(a, al, s);
  if (c.type == IC_BF16) return dw_typed<bf16_t>(a, al, s);
  return dw_typed<f16_t>(a, al, s);
}

}  // namespace ic
