// Log probabilities of labels over rows of scores, their entropy and best alternatives, and the
// gradient of the first two.
//
// With z_j = x_j / T for the V scores of a row:
//     M = max_j x_j,   s = sum_j e^{(x_j - M)/T},   u = sum_j e^{(x_j - M)/T} (x_j - M)
//     lse = M/T + ln s,   log p_j = (x_j - M)/T - ln s,   H = -sum_j p_j log p_j = ln s - u/(T s)
// so one pass over the row gives everything: (M, s, u) of two pieces of a row join as
//     M = max(M1, M2),  s = s1 f1 + s2 f2,  u = (u1 + s1 (M1 - M)) f1 + ...,  f = e^{(M1 - M)/T}.
// Both terms of H are >= 0, so a peaked row's small entropy does not come out of a cancellation.
// All sums are float32 over float32 terms, added as a tree of 64 lanes x waves x pieces.
//
// Special rows: scores of -inf have p = 0 and add nothing (the product 0 * (x - M) is kept finite
// by clamping x - M); a row of nothing but -inf has lse = -inf, H = 0, log p = -inf and gradient 0;
// a row with NaN or +inf has NaN results (its alternatives are still ranked, NaN above +inf).
//
// The best alternatives: values are ranked as integers (a monotone map of the float bits, -0 as
// +0), ties to the lowest index.  A lane keeps its own two best while it streams; the t best of a
// wave are then t rounds of a 64-lane maximum, in which only the winner moves on.  Where a lane has
// given away both of its two, its part of the row is looked through again for what follows (and, where
// the row is in registers, every lane's for its best two of the rest: about every tenth round).
//
// What bounds it: reading the row once, and the instructions that rank it; the figures stand at each
// kernel.
#include <climits>

#include "ic_wave.h"

namespace ic {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kFar = -1.0e30f;      // x - M of a masked score: e^kFar is 0 and 0 * kFar is 0
constexpr float kGone = -128.0f;      // the same for log p: a probability that small is 0, and times any weight stays 0
constexpr float kLowest = -3.402823466e38f;

// monotone in the value, 0 below everything (an absent element)
__device__ __forceinline__ unsigned rank_of(float x) {
  const unsigned b = __float_as_uint(x + 0.0f);
  const unsigned k = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
  return x != x ? 0xffffffffu : k;
}
__device__ __forceinline__ float value_of(unsigned k) {
  return __uint_as_float((k & 0x80000000u) ? (k ^ 0x80000000u) : ~k);
}

struct Stats {
  float m, s, u;
};

__device__ __forceinline__ float gap(float x, float m) { return fmaxf(x - m, kFar); }

// c = log2(e) / T
__device__ __forceinline__ void rescale(Stats& a, float m, float c) {
  const float d = gap(a.m, m);
  const float f = __builtin_amdgcn_exp2f(d * c);
  a.u = (a.u + a.s * d) * f;
  a.s *= f;
  a.m = m;
}

template <int N>
__device__ __forceinline__ void add_values(Stats& a, const float* x, float c) {
  float vm = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) vm = fmaxf(vm, x[i]);
  rescale(a, fmaxf(a.m, vm), c);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float d = x[i] - a.m;
    const float e = __builtin_amdgcn_exp2f(d * c);   // NaN for NaN and for +inf: s carries it on
    a.s += e;
    a.u = fmaf(e, fmaxf(d, kFar), a.u);
  }
}

// the 64 lanes' pieces as one, in every lane
__device__ __forceinline__ Stats wave_join(Stats a, float c) {
  rescale(a, wave_max_f32(a.m), c);
  a.s = wave_sum_f32(a.s);
  a.u = wave_sum_f32(a.u);
  return a;
}

// A lane's two best: (rank, index) descending by rank, ascending by index.
struct Best2 {
  unsigned k1, k2;
  int i1, i2;
};
__device__ __forceinline__ void keep(Best2& b, unsigned k, int i) {   // i ascends within a lane
  const bool first = k > b.k1, second = k > b.k2;
  b.i2 = first ? b.i1 : (second ? i : b.i2);
  b.k2 = first ? b.k1 : (second ? k : b.k2);
  b.i1 = first ? i : b.i1;
  b.k1 = first ? k : b.k1;
}
__device__ __forceinline__ bool after(unsigned k, int i, unsigned k0, int i0) {
  return k < k0 || (k == k0 && i > i0);
}

// The lane that holds the best (rank, index) of all lanes' heads.
__device__ __forceinline__ int best_lane(unsigned k, int i, unsigned* kb) {
  const unsigned top = wave_max_u32(k);
  *kb = top;
  unsigned long long who = __ballot(k == top);
  if (who & (who - 1)) {   // equal values: the lowest index
    const unsigned low = wave_min_u32(k == top ? (unsigned)i : 0xffffffffu);
    who = __ballot(k == top && (unsigned)i == low);
  }
  return __builtin_amdgcn_readfirstlane(__ffsll(who) - 1);
}

// t rounds over the lanes' lists; lane r returns with the r-th best.  refill(w, k, i, b, left), called where
// lane w has given away both of its two, brings the lists up to date with (k, i) taken last.
template <typename Refill>
__device__ __forceinline__ void take_best(Best2 b, int t, int lane, unsigned* out_k, int* out_i,
                                          Refill refill) {
  int left = 2;
  unsigned rk = 0;
  int ri = -1;
  for (int r = 0; r < t; ++r) {
    unsigned kb;
    const int w = best_lane(b.k1, b.i1, &kb);
    const int ib = __builtin_amdgcn_readlane(b.i1, w);
    if (lane == r) {
      rk = kb;
      ri = ib;
    }
    if (lane == w) {
      b.k1 = b.k2;
      b.i1 = b.i2;
      b.k2 = 0;
      --left;
    }
    if (r + 1 < t && __builtin_amdgcn_readlane(left, w) == 0) {
      refill(w, kb, ib, &b, &left);
    }
  }
  *out_k = rk;
  *out_i = ri;
}

// Where a row lies: granules of 16 aligned bytes from the one that holds its first element on; a
// granule that the row fills is loaded whole, one at either end of the row element by element.
template <typename T>
struct RowView {
  const T* row;
  const char* base;   // row rounded down to 16 bytes
  int head;           // elements of the first granule that lie before the row
  int v;
  __device__ RowView(const T* r, int v_) : row(r), v(v_) {
    const uintptr_t a = reinterpret_cast<uintptr_t>(r);
    base = reinterpret_cast<const char*>(a & ~(uintptr_t)15);
    head = (int)((a & 15) / sizeof(T));
  }
  __device__ __forceinline__ int granules() const {
    return (v + head + Elem<T>::kVec - 1) / Elem<T>::kVec;
  }
  // elements g * kVec - head .. of the row, -inf outside it
  __device__ __forceinline__ u32x4 get_raw(int g) const {
    constexpr int kV = Elem<T>::kVec;
    const int j0 = g * kV - head;
    if (j0 >= 0 && j0 + kV <= v) return *reinterpret_cast<const u32x4*>(base + (size_t)g * 16);
    float x[kV];
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const int j = j0 + i;
      x[i] = (j >= 0 && j < v) ? Elem<T>::load(row + j) : -__builtin_inff();
    }
    return Elem<T>::pack(x);
  }
  __device__ __forceinline__ void get(int g, float* x) const { Elem<T>::unpack(get_raw(g), x); }
};

struct ScoreArgs {
  const void* logits;
  int64_t ld;
  int64_t row0, n;      // rows [row0, n) are this launch's
  int v;
  const void* labels;   // int32 or int64
  int labels64;
  float inv_t;
  int top;
  float* logp;
  float* entropy;
  float* lse;
  float* top_logp;
  int32_t* top_idx;
};

__device__ __forceinline__ int label_of(const ScoreArgs& a, int64_t row) {
  if (!a.labels) return -1;
  const int64_t l = a.labels64 ? static_cast<const int64_t*>(a.labels)[row]
                               : (int64_t) static_cast<const int32_t*>(a.labels)[row];
  return l >= 0 && l < a.v ? (int)l : -1;
}

// One lane writes the row's results; lanes 0 .. top-1 its alternatives.
template <typename T>
__device__ __forceinline__ void write_row(const ScoreArgs& a, int64_t row, const T* x, Stats st,
                                          int lane, unsigned rk, int ri) {
  const bool none = st.s == 0.0f;   // nothing but -inf
  const float ln_s = __builtin_amdgcn_logf(st.s) * kLn2;
  if (lane == 0) {
    a.lse[row] = none ? -__builtin_inff() : fmaf(st.m, a.inv_t, ln_s);
    a.entropy[row] = none ? 0.0f : fmaxf(ln_s - st.u * a.inv_t / st.s, 0.0f) + 0.0f * st.s;
    if (a.logp) {
      const int l = label_of(a, row);
      float lp = 0.0f;
      if (l >= 0) {
        const float z = Elem<T>::load(x + l);
        lp = none ? -__builtin_inff() : (z - st.m) * a.inv_t - ln_s;
      }
      a.logp[row] = lp;
    }
  }
  if (lane < a.top) {
    const float z = value_of(rk);
    a.top_idx[row * a.top + lane] = ri;
    a.top_logp[row * a.top + lane] = none ? -__builtin_inff() : (z - st.m) * a.inv_t - ln_s;
  }
}

// 16-bit scores of a row of at most kPackedMost columns rank as one 32-bit word: the monotone 16 bits
// of the score above, 65535 - index below.  All words differ, so ranking is minima and maxima of words,
// ties included, and an element behind the row (-inf, a larger index) never comes before one of the
// row.  NaN does not rank this way: rows that hold one take the general path.
constexpr int kPackedMost = 65520;
template <typename T>
__device__ __forceinline__ unsigned rank16x2(unsigned w) {   // two scores, -0 as +0
  typedef short s16x2 __attribute__((ext_vector_type(2)));
  const s16x2 v = __builtin_bit_cast(s16x2, w);
  const s16x2 sign = v >> (short)15;
  const s16x2 mag = v & (short)0x7fff;
  const s16x2 k = ((mag ^ sign) - sign) ^ (short)0x8000;
  return __builtin_bit_cast(unsigned, k);
}
template <typename T> __device__ __forceinline__ float value16(unsigned key16);
template <> __device__ __forceinline__ float value16<bf16_t>(unsigned k) {
  const unsigned b = (k & 0x8000u) ? k ^ 0x8000u : 0x8000u | (0x8000u - k);
  return __uint_as_float(b << 16);
}
template <> __device__ __forceinline__ float value16<f16_t>(unsigned k) {
  const unsigned b = (k & 0x8000u) ? k ^ 0x8000u : 0x8000u | (0x8000u - k);
  return (float)__builtin_bit_cast(_Float16, (unsigned short)b);
}
template <> __device__ __forceinline__ float value16<float>(unsigned) { return 0.0f; }

// Rows of up to 64 * NC granules: one wave a row, the row stays in registers between the maximum,
// the sums and the ranking.  100 000 rows of 1000 bf16 scores with the best five: 69 to 74 us, 2.9 TB/s: bound by
// its vector instructions (reading the row is 40 us; ranked as 32-bit words with an index each 111 us).
template <typename T, int NC, bool TOP>
__global__ __launch_bounds__(256) void k_score_wave(ScoreArgs a) {
  constexpr int kV = Elem<T>::kVec;
  const int lane = threadIdx.x & 63;
  const int64_t row = a.row0 + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.n) return;
  const T* xr = static_cast<const T*>(a.logits) + row * a.ld;
  const RowView<T> rv(xr, a.v);
  const float c = a.inv_t * kLog2e;
  u32x4 raw[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) raw[i] = rv.get_raw(i * 64 + lane);
  float m = kLowest;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float x[kV];
    Elem<T>::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < kV; ++j) m = fmaxf(m, x[j]);
  }
  Stats st;
  st.m = wave_max_f32(m);
  st.s = 0.0f;
  st.u = 0.0f;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    float x[kV];
    Elem<T>::unpack(raw[i], x);
#pragma unroll
    for (int j = 0; j < kV; ++j) {
      const float d = x[j] - st.m;
      const float e = __builtin_amdgcn_exp2f(d * c);
      st.s += e;
      st.u = fmaf(e, fmaxf(d, kFar), st.u);
    }
  }
  st.s = wave_sum_f32(st.s);
  st.u = wave_sum_f32(st.u);
  unsigned rk = 0;
  int ri = -1;
  if (TOP) {
    if (sizeof(T) == 2 && a.v <= kPackedMost && st.s == st.s) {
      // word (i, w, h): element 2 w + h of granule i.  Unless `all`, only words below floor_ count.
      auto best2 = [&](bool all, unsigned floor_, unsigned* k1, unsigned* k2) {
        unsigned b1 = 0, b2 = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          const int low = 65535 - ((i * 64 + lane) * kV - rv.head);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const unsigned pair = rank16x2<T>(raw[i][w]);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const unsigned at = (unsigned)(low - 2 * w - h);
              unsigned k = h ? (pair & 0xffff0000u) | (at & 0xffffu) : (pair << 16) | (at & 0xffffu);
              // (elements before the row lie in granule 0)
              if (i == 0 && rv.head) k = at > 65535u ? 0u : k;
              if (!all) k = k < floor_ ? k : 0u;
              // the median of the best two and a third is the new second
              asm("v_med3_u32 %0, %1, %2, %3" : "=v"(b2) : "v"(b1), "v"(b2), "v"(k));
              b1 = b1 > k ? b1 : k;
            }
          }
        }
        *k1 = b1;
        *k2 = b2;
      };
      unsigned k1, k2;
      best2(true, 0u, &k1, &k2);
      unsigned mine = 0;
      for (int r = 0; r < a.top; ++r) {
        const unsigned kb = wave_max_u32(k1);
        mine = lane == r ? kb : mine;
        const bool won = k1 == kb;
        // where a lane gives away its second, all look for their best two of what is left
        const bool spent = won && k2 == 0u;
        k1 = won ? k2 : k1;
        k2 = won ? 0u : k2;
        if (r + 1 < a.top && __ballot(spent)) {
          unsigned n1, n2;
          best2(false, kb, &n1, &n2);
          k1 = n1;
          k2 = n2;
        }
      }
      ri = 65535 - (int)(mine & 0xffffu);
      rk = rank_of(value16<T>(mine >> 16));
    } else {
      auto index_at = [&](int i, int j) { return (i * 64 + lane) * kV + j - rv.head; };
      auto inside = [&](int idx) { return idx >= 0 && idx < a.v; };
      auto best2 = [&](unsigned k0, int i0, bool all) {
        Best2 q = {0u, 0u, -1, -1};
#pragma unroll
        for (int i = 0; i < NC; ++i) {
          // (16 bits: rows with NaN.  Opaque: unpacked here, not kept in registers from the sums on, which
          // would cost the usual path its waves)
          u32x4 own = raw[i];
          if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(own));
          float x[kV];
          Elem<T>::unpack(own, x);
#pragma unroll
          for (int j = 0; j < kV; ++j) {
            const int idx = index_at(i, j);
            const unsigned k = inside(idx) ? rank_of(x[j]) : 0u;
            if (all || after(k, idx, k0, i0)) keep(q, k, idx);
          }
        }
        return q;
      };
      take_best(best2(0u, 0, true), a.top, lane, &rk, &ri, [&](int, unsigned k0, int i0, Best2* b, int* left) {
        *b = best2(k0, i0, false);     // all lanes' best two of what is left
        *left = 2;
      });
    }
  }
  write_row<T>(a, row, xr, st, lane, rk, ri);
}

// Rows of up to 64 scores: 2^LOG lanes a row, a score a lane, so that a wave takes up to 16 rows; what a
// row's lanes reduce is left in all of them.
template <int X>
__device__ __forceinline__ unsigned from_lane_xor(unsigned v) {
  if constexpr (X == 1) return dpp_u32<0xb1>(v, v);                     // quad_perm 1 0 3 2
  else if constexpr (X == 2) return dpp_u32<0x4e>(v, v);                // quad_perm 2 3 0 1
  else if constexpr (X == 4) {
    const unsigned w = dpp_u32<0x141>(v, v);                            // row_half_mirror: xor 7
    return dpp_u32<0x1b>(w, w);                                         // quad_perm 3 2 1 0: xor 3
  } else if constexpr (X == 8) return dpp_u32<0x128>(v, v);             // row_ror 8
  else return (unsigned)__shfl_xor((int)v, X, 64);
}
__device__ __forceinline__ uint64_t pair64(unsigned high, unsigned low) { return (uint64_t)high << 32 | low; }
template <int X>
__device__ __forceinline__ uint64_t from_lane_xor(uint64_t v) {
  return pair64(from_lane_xor<X>((unsigned)(v >> 32)), from_lane_xor<X>((unsigned)v));
}
template <int X, int L, typename F>
__device__ __forceinline__ float lanes_fold(float v, F op) {
  if constexpr (X < L) {
    v = op(v, __uint_as_float(from_lane_xor<X>(__float_as_uint(v))));
    return lanes_fold<2 * X, L>(v, op);
  } else {
    return v;
  }
}
// Bitonic sort of the keys of L lanes, descending: blocks of K lanes, partners J apart.
template <int K, int J, int L, typename Key>
__device__ __forceinline__ Key lanes_sort(Key k, int lane) {
  if constexpr (K > L) {
    return k;
  } else {
    const Key other = from_lane_xor<J>(k);
    const bool larger = ((lane & J) == 0) == ((lane & K) == 0 || K == L);
    k = (k > other) == larger ? k : other;     // (equal keys: either)
    if constexpr (J > 1) return lanes_sort<K, J / 2, L>(k, lane);
    else return lanes_sort<2 * K, K, L>(k, lane);
  }
}

// Bound by instructions and, up to a few thousand rows, by latency: 54 184 rows of 18 bf16 scores with the best
// eleven 14 us (a wave a row 58), 50 000 rows of 60 float32 with the best thirty 28 us (99).
template <typename T, int LOG, bool TOP>
__global__ __launch_bounds__(256) void k_score_small(ScoreArgs a) {
  constexpr int L = 1 << LOG;
  const int lane = threadIdx.x & 63, sub = lane & (L - 1);
  int64_t row = a.row0 + (int64_t)blockIdx.x * (256 / L) + (threadIdx.x >> LOG);
  const bool ours = row < a.n;
  if (!ours) row = a.n - 1;          // (its lanes take part and write nothing)
  const T* xr = static_cast<const T*>(a.logits) + row * a.ld;
  const bool in = sub < a.v;
  const float x = in ? Elem<T>::load(xr + sub) : -__builtin_inff();
  const float c = a.inv_t * kLog2e;
  auto most = [](float p, float q) { return fmaxf(p, q); };
  auto sum = [](float p, float q) { return p + q; };
  Stats st;
  st.m = lanes_fold<1, L>(fmaxf(x, kLowest), most);
  const float d = x - st.m;
  const float e = __builtin_amdgcn_exp2f(d * c);
  st.s = lanes_fold<1, L>(e, sum);
  st.u = lanes_fold<1, L>(e * fmaxf(d, kFar), sum);
  unsigned rk = 0;
  int ri = -1;
  if constexpr (TOP) {
    // keys differ, ties rank by index; lanes behind the row come last
    if constexpr (sizeof(T) == 2) {
      const unsigned bits = reinterpret_cast<const unsigned short*>(xr)[in ? sub : 0];
      const unsigned r16 = x != x ? 0xffffu : rank16x2<T>(bits) & 0xffffu;
      const unsigned key = lanes_sort<2, 1, L>(in ? r16 << 16 | (unsigned)(65535 - sub) : 0u, lane);
      ri = 65535 - (int)(key & 0xffffu);
      rk = rank_of(value16<T>(key >> 16));
    } else {
      const uint64_t key = lanes_sort<2, 1, L>(in ? pair64(rank_of(x), 0xffffffffu - (unsigned)sub) : (uint64_t)0, lane);
      ri = (int)(0xffffffffu - (unsigned)key);
      rk = (unsigned)(key >> 32);
    }
  }
  if (ours) write_row<T>(a, row, xr, st, sub, rk, ri);
}

// A piece of a row as k_score_pieces leaves it: 4 words, then top (rank, index) pairs
__host__ __device__ inline size_t piece_words(int top) { return 4 + 2 * (size_t)top; }

constexpr int kPieceThreads = 256;
constexpr int kPieceWaves = kPieceThreads / 64;

// Longer rows: a workgroup streams one of `pieces` pieces of a row (pieces > 1 where there are too
// few rows to fill the card; k_score_join then joins them).  4096 rows of 65 536 bf16 scores: 125 to 138 us,
// 3.9 to 4.3 TB/s (a sum over 1 GiB by the library reads 3.9), 103 us where the last level cache still holds a
// part of them; 8 rows of 65 536 float32 scores with the
// best ten: 8.8 us and 4.6 for the join, latency.
template <typename T, bool TOP>
__global__ __launch_bounds__(kPieceThreads) void k_score_pieces(ScoreArgs a, int pieces,
                                                                unsigned* part) {
  constexpr int kV = Elem<T>::kVec;
  __shared__ float sm[kPieceWaves][4];
  __shared__ unsigned lk[kPieceWaves][32];
  __shared__ int li[kPieceWaves][32];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = a.row0 + blockIdx.x;
  const int piece = blockIdx.y;
  const T* xr = static_cast<const T*>(a.logits) + row * a.ld;
  const RowView<T> rv(xr, a.v);
  const float c = a.inv_t * kLog2e;
  const int64_t total = rv.granules();
  const int g0 = (int)(total * piece / pieces), g1 = (int)(total * (piece + 1) / pieces);
  Stats st = {kLowest, 0.0f, 0.0f};
  Best2 b = {0u, 0u, -1, -1};
  auto take = [&](const float* x, int g) {
    if (TOP) {
      const int j0 = g * kV - rv.head;
#pragma unroll
      for (int j = 0; j < kV; ++j) {
        const int idx = j0 + j;
        keep(b, idx >= 0 && idx < a.v ? rank_of(x[j]) : 0u, idx);
      }
    }
  };
  int g = g0 + (int)threadIdx.x;
  // two granules per lane and step: their loads are in flight together
  for (; g + kPieceThreads < g1; g += 2 * kPieceThreads) {
    float x[2 * kV];
    rv.get(g, x);
    rv.get(g + kPieceThreads, x + kV);
    add_values<2 * kV>(st, x, c);
    take(x, g);
    take(x + kV, g + kPieceThreads);
  }
  if (g < g1) {
    float x[kV];
    rv.get(g, x);
    add_values<kV>(st, x, c);
    take(x, g);
  }
  st = wave_join(st, c);
  if (lane == 0) {
    sm[wave][0] = st.m;
    sm[wave][1] = st.s;
    sm[wave][2] = st.u;
  }
  if (TOP) {
    unsigned rk;
    int ri;
    const int t0 = g0 + (wave << 6);
    take_best(b, a.top, lane, &rk, &ri, [&](int w, unsigned k0, int i0, Best2* lists, int* left) {
      // lane w's granules are t0 + w, + kPieceThreads, ...: the 64 lanes look through them
      Best2 q = {0u, 0u, -1, -1};
      for (int64_t h = (int64_t)t0 + w + (int64_t)lane * kPieceThreads; h < g1;
           h += 64 * kPieceThreads) {
        float x[kV];
        rv.get((int)h, x);
        const int j0 = (int)h * kV - rv.head;
#pragma unroll
        for (int j = 0; j < kV; ++j) {
          const int idx = j0 + j;
          const unsigned k = idx >= 0 && idx < a.v ? rank_of(x[j]) : 0u;
          if (after(k, idx, k0, i0)) keep(q, k, idx);
        }
      }
      unsigned kb;
      const int from = best_lane(q.k1, q.i1, &kb);
      const int ib = __builtin_amdgcn_readlane(q.i1, from);
      if (lane == w) {
        lists->k1 = kb;
        lists->i1 = ib;
        *left = 1;
      }
    });
    if (lane < a.top) {
      lk[wave][lane] = rk;
      li[wave][lane] = ri;
    }
  }
  __syncthreads();
  if (wave != 0) return;
  Stats j = {kLowest, 0.0f, 0.0f};
  if (lane < kPieceWaves) {
    j.m = sm[lane][0];
    j.s = sm[lane][1];
    j.u = sm[lane][2];
  }
  j = wave_join(j, c);
  unsigned rk = 0;
  int ri = -1;
  if (TOP) {
    // lane w walks wave w's list
    int at = 0;
    unsigned k = lane < kPieceWaves ? lk[lane][0] : 0u;
    int i = lane < kPieceWaves ? li[lane][0] : 0x7fffffff;
    for (int r = 0; r < a.top; ++r) {
      unsigned kb;
      const int w = best_lane(k, i, &kb);
      const int ib = __builtin_amdgcn_readlane(i, w);
      if (lane == r) {
        rk = kb;
        ri = ib;
      }
      if (lane == w) {
        ++at;
        k = at < a.top ? lk[w][at] : 0u;
        i = at < a.top ? li[w][at] : 0x7fffffff;
      }
    }
  }
  if (pieces == 1) {
    write_row<T>(a, row, xr, j, lane, rk, ri);
    return;
  }
  unsigned* out = part + ((size_t)row * pieces + piece) * piece_words(a.top);
  if (lane == 0) {
    out[0] = __float_as_uint(j.m);
    out[1] = __float_as_uint(j.s);
    out[2] = __float_as_uint(j.u);
  }
  if (lane < a.top) {
    out[4 + 2 * lane] = rk;
    out[5 + 2 * lane] = (unsigned)ri;
  }
}

// One wave a row: lane p holds piece p (at most 64 pieces).
template <typename T>
__global__ __launch_bounds__(64) void k_score_join(ScoreArgs a, int pieces, const unsigned* part) {
  const int lane = threadIdx.x;
  const int64_t row = a.row0 + blockIdx.x;
  const T* xr = static_cast<const T*>(a.logits) + row * a.ld;
  const bool mine = lane < pieces;
  const unsigned* in = part + ((size_t)row * pieces + (mine ? lane : 0)) * piece_words(a.top);
  Stats j = {kLowest, 0.0f, 0.0f};
  if (mine) {
    j.m = __uint_as_float(in[0]);
    j.s = __uint_as_float(in[1]);
    j.u = __uint_as_float(in[2]);
  }
  j = wave_join(j, a.inv_t * kLog2e);
  unsigned rk = 0;
  int ri = -1;
  int at = 0;
  unsigned k = mine && a.top > 0 ? in[4] : 0u;
  int i = mine && a.top > 0 ? (int)in[5] : 0x7fffffff;
  for (int r = 0; r < a.top; ++r) {
    unsigned kb;
    const int w = best_lane(k, i, &kb);
    const int ib = __builtin_amdgcn_readlane(i, w);
    if (lane == r) {
      rk = kb;
      ri = ib;
    }
    if (lane == w) {
      ++at;
      k = at < a.top ? in[4 + 2 * at] : 0u;
      i = at < a.top ? (int)in[5 + 2 * at] : 0x7fffffff;
    }
  }
  write_row<T>(a, row, xr, j, lane, rk, ri);
}

struct GradArgs {
  const void* logits;
  int64_t ld;
  int64_t row0, n;
  int v;
  const void* labels;
  int labels64;
  float inv_t;
  const float* lse;
  const float* entropy;
  const float* d_logp;      // may be NULL: no gradient through log p
  const float* d_entropy;   // may be NULL
  void* out;
  int64_t ld_out;
};

// p_j = e^(x_j / T - lse) is as good as lse is: rounded to float32 it is off by half its last bit, and p by as
// much of itself.  Up to this size that is 2^-20 (float32 scores), and 2^-17 where p is rounded to 2^-9 or 2^-12
// afterwards.  Beyond it (all scores of a row shifted far from zero, rows masked with the type's lowest value)
// the row is "far": its maximum M and ln s are worked out once more, and log p = (x - M) / T - ln s as in
// the pass over the scores.
template <typename T>
__device__ __forceinline__ bool far_from_zero(float lse) {
  return fabsf(lse) > (sizeof(T) == 4 ? 32.0f : 256.0f);   // (and infinite; NaN is not)
}
// (M, s) of a row from its scores, in all of the row's lanes: lane `sub` of `lanes`, which are part of a wave or
// the whole workgroup (in which every row is far, then).
template <typename T, int THREADS>
__device__ __forceinline__ Stats row_again(const RowView<T>& rv, int total, int sub, int lanes, float c) {
  constexpr int kV = Elem<T>::kVec;
  __shared__ float sm[THREADS / 64], ss[THREADS / 64];
  Stats st = {kLowest, 0.0f, 0.0f};
  for (int q = sub; q < total; q += lanes) {
    float x[kV];
    rv.get(q, x);
    add_values<kV>(st, x, c);
  }
  const int within = lanes < 64 ? lanes : 64;
  float m = st.m;
  for (int o = 1; o < within; o <<= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  rescale(st, m, c);
  for (int o = 1; o < within; o <<= 1) st.s += __shfl_xor(st.s, o, 64);
  if (lanes > 64) {
    if ((threadIdx.x & 63) == 0) {
      sm[threadIdx.x >> 6] = st.m;
      ss[threadIdx.x >> 6] = st.s;
    }
    __syncthreads();   // (and no score is overwritten before all of the row have been read)
    for (int w = 0; w < THREADS / 64; ++w) m = fmaxf(m, sm[w]);
    st.m = m;
    st.s = 0.0f;
    for (int w = 0; w < THREADS / 64; ++w) st.s += ss[w] * __builtin_amdgcn_exp2f(gap(sm[w], m) * c);
  }
  return st;
}

// dL/dx_j = ( g (delta_{j,label} - p_j) - h p_j (log p_j + H) ) / T with g = dL/dlogp (0 for a row
// without a label) and h = dL/dH, for granules [g0, g1) of a row, by lane `sub` of `lanes`.  One read of the scores
// (two where `again`: the row is far), one write of the gradient (out may be the scores themselves: an element is
// read before it is written, by the same lane).
template <typename T, bool STREAM, int THREADS>
__device__ __forceinline__ void grad_row(const GradArgs& a, int64_t row, float lse, bool again, int sub, int lanes,
                                         int g0, int span) {
  constexpr int kV = Elem<T>::kVec;
  const T* xr = static_cast<const T*>(a.logits) + row * a.ld;
  T* yr = static_cast<T*>(a.out) + row * a.ld_out;
  int64_t l = -1;
  if (a.labels && a.d_logp)
    l = a.labels64 ? static_cast<const int64_t*>(a.labels)[row]
                   : (int64_t) static_cast<const int32_t*>(a.labels)[row];
  const int label = l >= 0 && l < a.v ? (int)l : -1;
  const float g = label >= 0 ? a.d_logp[row] : 0.0f;
  const float h = a.d_entropy ? a.d_entropy[row] : 0.0f;
  const float H = a.d_entropy ? a.entropy[row] : 0.0f;
  const RowView<T> rv(xr, a.v);
  const int total = rv.granules();
  const int g1 = total - g0 < span ? total : g0 + span;
  float m0 = 0.0f, l0 = lse;           // log p = (x - m0) / T - l0
  bool none = false;                   // nothing but -inf
  if (again) {
    const Stats st = row_again<T, THREADS>(rv, total, sub, lanes, a.inv_t * kLog2e);
    none = st.s == 0.0f;
    m0 = st.m;
    l0 = none ? 0.0f : __builtin_amdgcn_logf(st.s) * kLn2;
  }
  // the output row starts at the same place of a granule as the input row
  const bool same = (reinterpret_cast<uintptr_t>(yr) & 15) == (reinterpret_cast<uintptr_t>(xr) & 15);
  char* yb = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(yr) & ~(uintptr_t)15);
  for (int q = g0 + sub; q < g1; q += lanes) {
    float x[kV];
    rv.get(q, x);
    const int j0 = q * kV - rv.head;
#pragma unroll
    for (int i = 0; i < kV; ++i) {
      const float lq = fmaxf(fmaf(x[i] - m0, a.inv_t, -l0), kGone) + 0.0f * l0;
      const float p = __builtin_amdgcn_exp2f(lq * kLog2e);
      float d = -p * fmaf(h, lq + H, g);
      d = (j0 + i == label ? d + g : d) * a.inv_t;
      x[i] = none ? 0.0f : d;
    }
    if (same && j0 >= 0 && j0 + kV <= a.v) {
      u32x4* to = reinterpret_cast<u32x4*>(yb + (size_t)q * 16);
      if (STREAM) __builtin_nontemporal_store(Elem<T>::pack(x), to);
      else *to = Elem<T>::pack(x);
    } else {
#pragma unroll
      for (int i = 0; i < kV; ++i)
        if (j0 + i >= 0 && j0 + i < a.v) Elem<T>::store(yr + j0 + i, x[i]);
    }
  }
}

// Whole rows: 2^lanes_log2 lanes of a wave a row, or a workgroup.  Rows are taken from the last to the first, here
// and below: what the pass over the scores read last may still be in the last level cache (4096 rows of 65 536 bf16
// scores, 324 -> 317 us for both passes).  STREAM, for gradients that cache cannot hold: stores that do not push the
// scores out of it (-> 298 us when both passes are repeated over the same scores).
template <typename T, bool STREAM, int THREADS>
__global__ __launch_bounds__(THREADS) void k_score_grad(GradArgs a, int lanes_log2) {
  constexpr int kThreadsLog2 = THREADS == 1024 ? 10 : 8;
  const int lanes = 1 << lanes_log2;
  const int64_t row = a.row0 + ((int64_t)(gridDim.x - 1 - blockIdx.x) << (kThreadsLog2 - lanes_log2)) +
                      (threadIdx.x >> lanes_log2);
  if (row >= a.n) return;
  const float lse = a.lse[row];
  grad_row<T, STREAM, THREADS>(a, row, lse, far_from_zero<T>(lse), (int)threadIdx.x & (lanes - 1), lanes, 0, INT_MAX);
}

// Long rows in pieces of `span` granules, a workgroup each.  It leaves far rows to k_score_grad_far, in a launch behind
// it: none of several workgroups could read a row that the others already write to.  4096 rows of 65 536 bf16
// scores: bound by memory; 190 to 209 us, 5.1 to 5.7 TB/s (a copy of 1 GiB: 5.2), by what the last level cache holds.
template <typename T, bool STREAM>
__global__ __launch_bounds__(256) void k_score_grad_near(GradArgs a, int span) {
  const int64_t row = a.row0 + (gridDim.x - 1 - blockIdx.x);
  const float lse = a.lse[row];
  if (far_from_zero<T>(lse)) return;
  grad_row<T, STREAM, 256>(a, row, lse, false, threadIdx.x, 256, (int)blockIdx.y * span, span);
}

// The far rows among the long ones: a workgroup looks at every gridDim.x-th row, 64 at a time.
template <typename T, bool STREAM>
__global__ __launch_bounds__(1024) void k_score_grad_far(GradArgs a) {
  for (int64_t row0 = a.row0 + blockIdx.x; row0 < a.n; row0 += 64 * (int64_t)gridDim.x) {
    const int64_t mine = row0 + (threadIdx.x & 63) * (int64_t)gridDim.x;
    const float lse = mine < a.n ? a.lse[mine] : 0.0f;
    unsigned long long far = __ballot(far_from_zero<T>(lse));   // (the same in every wave)
    while (far) {
      const int64_t row = row0 + (__ffsll(far) - 1) * (int64_t)gridDim.x;
      far &= far - 1;
      grad_row<T, STREAM, 1024>(a, row, 0.0f, true, threadIdx.x, 1024, 0, INT_MAX);
      __syncthreads();   // (row_again's LDS is free)
    }
  }
}

// rows of one launch: the launch's threads are counted in 32 bits
constexpr int64_t kRowsPerLaunch = (int64_t)1 << 22;

// So many rows fill the card with a wave each.
constexpr int64_t kManyRows = 2048;

template <typename T, bool TOP>
hipError_t score_launch(ScoreArgs a, int pieces, unsigned* part, hipStream_t s) {
  // the longest row a wave keeps in registers: 8 granules a lane (one more than the row's length
  // asks for, because a row may start inside a granule)
  const int64_t granules = ((int64_t)a.v + 2 * Elem<T>::kVec - 2) / Elem<T>::kVec;
  const int64_t n = a.n;
  for (a.row0 = 0; a.row0 < n; a.row0 += kRowsPerLaunch) {
    const int64_t rows = n - a.row0 < kRowsPerLaunch ? n - a.row0 : kRowsPerLaunch;
    a.n = a.row0 + rows;
    const dim3 by4((unsigned)((rows + 3) / 4));
    if (a.v <= 64) {
      int log2 = 2;
      while ((1 << log2) < a.v) ++log2;
      const dim3 by((unsigned)((rows + (256 >> log2) - 1) / (256 >> log2)));
      switch (log2) {
        case 2: hipLaunchKernelGGL((k_score_small<T, 2, TOP>), by, dim3(256), 0, s, a); break;
        case 3: hipLaunchKernelGGL((k_score_small<T, 3, TOP>), by, dim3(256), 0, s, a); break;
        case 4: hipLaunchKernelGGL((k_score_small<T, 4, TOP>), by, dim3(256), 0, s, a); break;
        case 5: hipLaunchKernelGGL((k_score_small<T, 5, TOP>), by, dim3(256), 0, s, a); break;
        default: hipLaunchKernelGGL((k_score_small<T, 6, TOP>), by, dim3(256), 0, s, a); break;
      }
    } else if (granules <= 64) {
      hipLaunchKernelGGL((k_score_wave<T, 1, TOP>), by4, dim3(256), 0, s, a);
    } else if (granules <= 128) {
      hipLaunchKernelGGL((k_score_wave<T, 2, TOP>), by4, dim3(256), 0, s, a);
    } else if (granules <= 192) {
      hipLaunchKernelGGL((k_score_wave<T, 3, TOP>), by4, dim3(256), 0, s, a);
    } else if (granules <= 256) {
      hipLaunchKernelGGL((k_score_wave<T, 4, TOP>), by4, dim3(256), 0, s, a);
    } else if (granules <= 320) {
      hipLaunchKernelGGL((k_score_wave<T, 5, TOP>), by4, dim3(256), 0, s, a);
    } else if (granules <= 384) {
      hipLaunchKernelGGL((k_score_wave<T, 6, TOP>), by4, dim3(256), 0, s, a);
    } else if (granules <= 512) {
      hipLaunchKernelGGL((k_score_wave<T, 8, TOP>), by4, dim3(256), 0, s, a);
    } else if (TOP && sizeof(T) == 4 && granules <= 1024 && n >= kManyRows) {
      // (ranking by one wave instead of four and a join: 17 852 rows of 2151 with the best thirty 187 ->
      // 149 us, 20 000 of 4000 with the best five 94 -> 77; 16-bit rows of twice the length would need
      // 360 registers: 3000 rows of 5000 fp16, best sixteen, 34 -> 36 us)
      if constexpr (sizeof(T) == 4)
        hipLaunchKernelGGL((k_score_wave<T, 16, TOP>), by4, dim3(256), 0, s, a);
    } else {
      hipLaunchKernelGGL((k_score_pieces<T, TOP>), dim3((unsigned)rows, (unsigned)pieces),
                         dim3(kPieceThreads), 0, s, a, pieces, part);
      if (pieces > 1)
        hipLaunchKernelGGL(k_score_join<T>, dim3((unsigned)rows), dim3(64), 0, s, a, pieces, part);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, bool STREAM>
hipError_t grad_launch(GradArgs a, hipStream_t s) {
  const int64_t granules = ((int64_t)a.v + 2 * Elem<T>::kVec - 2) / Elem<T>::kVec;
  int lanes_log2 = 1;
  while (lanes_log2 < 8 && (1 << lanes_log2) < granules) ++lanes_log2;
  // (lanes of one wave, or the whole workgroup; 128 were slower anyway: 100 000 rows of 1000 bf16 74 -> 66 us)
  if (lanes_log2 == 7) lanes_log2 = 6;
  const int64_t n = a.n;
  const bool many = n >= kManyRows;
  // A workgroup a row while a lane has few granules of it; of 1024 lanes where there are few rows (1000 rows of 16 384
  // bf16: 13.0 us, with 256 lanes 14.5; 64 rows of 8192: 3.3, in pieces with the launch for the far ones 4.3)
  const bool whole = granules <= 4096;
  // else pieces (4096 rows of 65 536 bf16: 209 us, a workgroup a row 216) of 2048 granules, fewer when that leaves CUs
  // without work
  int64_t span = 2048;
  while (span > 256 && n * ((granules + span - 1) / span) < 8 * (int64_t)kCUs) span /= 2;
  while ((granules + span - 1) / span > 65535) span *= 2;
  for (a.row0 = 0; a.row0 < n; a.row0 += kRowsPerLaunch) {
    const int64_t rows = n - a.row0 < kRowsPerLaunch ? n - a.row0 : kRowsPerLaunch;
    a.n = a.row0 + rows;
    if (granules <= 256 || (whole && many)) {
      const int64_t per_wg = 256 >> lanes_log2;
      hipLaunchKernelGGL((k_score_grad<T, STREAM, 256>), dim3((unsigned)((rows + per_wg - 1) / per_wg)), dim3(256), 0,
                         s, a, lanes_log2);
    } else if (whole) {
      hipLaunchKernelGGL((k_score_grad<T, STREAM, 1024>), dim3((unsigned)rows), dim3(1024), 0, s, a, 10);
    } else {
      hipLaunchKernelGGL((k_score_grad_near<T, STREAM>), dim3((unsigned)rows, (unsigned)((granules + span - 1) / span)),
                         dim3(256), 0, s, a, (int)span);
      hipLaunchKernelGGL((k_score_grad_far<T, STREAM>), dim3((unsigned)(rows < 2 * kCUs ? rows : 2 * kCUs)), dim3(1024),
                         0, s, a);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T>
hipError_t grad_typed(const GradArgs& a, hipStream_t s) {
  // half of the last level cache: a smaller gradient is left there for who reads it next
  const bool stream = a.n * a.v > ((int64_t)128 << 20) / (int64_t)sizeof(T);
  return stream ? grad_launch<T, true>(a, s) : grad_launch<T, false>(a, s);
}

}  // namespace

int score_pieces(int64_t n, int64_t v, int dtype) {
  const int vec = dtype == IC_F32 ? 4 : 8;
  const int64_t granules = (v + 2 * vec - 2) / vec;
  if (granules <= 64 * 8 || n == 0) return 1;
  // four workgroups a CU, and at least two granules a lane in a piece
  int64_t p = (4 * (int64_t)kCUs + n - 1) / n;
  const int64_t most = granules / (2 * kPieceThreads);
  if (p > most) p = most;
  return (int)(p < 1 ? 1 : p > 64 ? 64 : p);
}

size_t score_scratch_bytes(int64_t n, int pieces, int top) {
  return pieces > 1 ? (size_t)n * pieces * piece_words(top) * 4 : 0;
}

hipError_t launch_label_logprobs(const void* logits, int dtype, int64_t ld, int64_t n, int64_t v,
                                 const void* labels, int labels64, float inv_t, int top, float* logp,
                                 float* entropy, float* lse, float* top_logp, int32_t* top_idx,
                                 int pieces, void* scratch, hipStream_t s) {
  const ScoreArgs a{logits, ld, 0, n, (int)v, labels, labels64, inv_t, top, logp, entropy, lse, top_logp,
                    top_idx};
  unsigned* part = static_cast<unsigned*>(scratch);
  if (dtype == IC_F32)
    return top ? score_launch<float, true>(a, pieces, part, s) : score_launch<float, false>(a, pieces, part, s);
  if (dtype == IC_BF16)
    return top ? score_launch<bf16_t, true>(a, pieces, part, s) : score_launch<bf16_t, false>(a, pieces, part, s);
  return top ? score_launch<f16_t, true>(a, pieces, part, s) : score_launch<f16_t, false>(a, pieces, part, s);
}

hipError_t launch_label_logprobs_grad(const void* logits, int dtype, int64_t ld, int64_t n, int64_t v,
                                      const void* labels, int labels64, float inv_t, const float* lse,
                                      const float* entropy, const float* d_logp,
                                      const float* d_entropy, void* out, int64_t ld_out, hipStream_t s) {
  const GradArgs a{logits, ld, 0, n, (int)v, labels, labels64, inv_t, lse, entropy, d_logp, d_entropy, out,
                   ld_out};
  if (dtype == IC_F32) return grad_typed<float>(a, s);
  if (dtype == IC_BF16) return grad_typed<bf16_t>(a, s);
  return grad_typed<f16_t>(a, s);
}

}  // namespace ic
