// One AdamW step over many tensors, with optimizer states in 32 or in 8 bits.
//
//     m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2
//     p <- p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// The tensors' addresses travel as kernel arguments, kTensorsPerLaunch a launch, so that a step is
// launches only: nothing is uploaded, and a captured graph holds the addresses it was captured with.
// States lie in flat arrays in which every tensor starts at a multiple of kStateBlock elements.
//
// States in 8 bits: kStateBlock elements share two float32 scales.
//   m: sign, 4-bit exponent, 3-bit mantissa of m / scale_m, with scale_m = max |m| / 448 (448 is
//      the largest finite code, 126; 127 marks a value that is not finite);
//   v: an unsigned 4-bit exponent, 4-bit mantissa code of sqrt(v) / scale_v, scale_v = max / 491520
//      (code 254; 255 marks a value that is not finite).  sqrt(v) rather than v: the step divides
//      by it, and its range is half as many octaves.  A state above zero keeps a code above zero,
//      so the step never divides by eps alone where a gradient was seen.
// Both roundings are to nearest, an exact middle to the even code, at most 2^-4 (m) and 2^-5
// (sqrt v) of the value, and the codes are decided in float64 (see k_adamw8): which of two codes a
// value takes then does not depend on the last bit of a float32 evaluation.  A scale that is a float32
// subnormal (a block's maximum below 6e-36 for m, 6e-33 for sqrt v) is itself off by up to a half, and what
// then lies above the largest code takes the largest code.
// The update uses the new m and v before they are rounded.
//
// What bounds it: memory with 32-bit states, instructions with 8-bit ones; the figures stand at each
// kernel.
#include <cmath>

#include "ic_wave.h"

namespace ic {

namespace {

struct AdamTable {
  AdamTensor t[kTensorsPerLaunch];
  int count;
};

struct AdamArgs {
  void* m;
  void* v;
  float* scale_m;
  float* scale_v;
  double lr, b1, b2, omb1, omb2, eps, wd, c1, c2;   // omb = 1 - b; c = 1 - b^t
  double lr1, root2;         // lr / c1, sqrt(1 / c2): the usual step has no division in the kernel
  const float* lr_dev;       // not NULL: the learning rate is read here
  const int64_t* step_dev;   // not NULL: t is read here; below 1 counts as 1
  float grad_scale;
};

constexpr int kChunk = 2048;   // elements of a workgroup's pass: 256 lanes x 8

__device__ __forceinline__ int find_tensor(const AdamTable& tab, int chunk) {
  int lo = 0, hi = tab.count;   // the last tensor whose chunk0 <= chunk
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (tab.t[mid].chunk0 <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

// b^t for t >= 0 by squaring
__device__ double power(double b, int64_t t) {
  double r = 1.0;
  for (; t > 0; t >>= 1) {
    if (t & 1) r *= b;
    b *= b;
  }
  return r;
}

// eight consecutive elements at p + i; those at and behind n are 0
template <typename T>
__device__ __forceinline__ void get8(const T* p, int64_t i, int64_t n, bool vec, float* x) {
  constexpr int kV = Elem<T>::kVec;
  if (vec && i + 8 <= n) {
#pragma unroll
    for (int q = 0; q < 8; q += kV) Elem<T>::unpack(*reinterpret_cast<const u32x4*>(p + i + q), x + q);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q) x[q] = i + q < n ? Elem<T>::load(p + i + q) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void put8(T* p, int64_t i, int64_t n, bool vec, const float* x) {
  constexpr int kV = Elem<T>::kVec;
  if (vec && i + 8 <= n) {
#pragma unroll
    for (int q = 0; q < 8; q += kV) *reinterpret_cast<u32x4*>(p + i + q) = Elem<T>::pack(x + q);
  } else {
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (i + q < n) Elem<T>::store(p + i + q, x[q]);
  }
}
__device__ __forceinline__ void get_typed(const void* p, int type, int64_t i, int64_t n, bool vec,
                                          float* x) {
  if (type == IC_F32) get8(static_cast<const float*>(p), i, n, vec, x);
  else if (type == IC_BF16) get8(static_cast<const bf16_t*>(p), i, n, vec, x);
  else get8(static_cast<const f16_t*>(p), i, n, vec, x);
}
__device__ __forceinline__ void put_typed(void* p, int type, int64_t i, int64_t n, bool vec,
                                          const float* x) {
  if (type == IC_F32) put8(static_cast<float*>(p), i, n, vec, x);
  else if (type == IC_BF16) put8(static_cast<bf16_t*>(p), i, n, vec, x);
  else put8(static_cast<f16_t*>(p), i, n, vec, x);
}

__device__ __forceinline__ void corrections(const AdamArgs& a, double* lr, double* lr1, double* root2) {
  *lr = a.lr;
  *lr1 = a.lr1;
  *root2 = a.root2;
  if (a.lr_dev || a.step_dev) {
    if (a.lr_dev) *lr = (double)*a.lr_dev;
    double c1 = a.c1;
    if (a.step_dev) {
      const int64_t t = *a.step_dev < 1 ? 1 : *a.step_dev;   // (counted from 1)
      c1 = 1.0 - power(a.b1, t);
      *root2 = sqrt(1.0 / (1.0 - power(a.b2, t)));
    }
    *lr1 = *lr / c1;
  }
}

// 256 lanes x 8 elements a workgroup.  64 Mi float32 parameters in 40 tensors: 342 us, 5.5 TB/s (a copy of
// 1 GiB: 5.2): bound by memory.  60 000 elements in 12 tensors: 5.4 us, latency.
__global__ __launch_bounds__(256) void k_adamw32(AdamTable tab, AdamArgs a) {
  const int chunk = blockIdx.x;
  const AdamTensor& t = tab.t[find_tensor(tab, chunk)];
  const int64_t i = (int64_t)(chunk - t.chunk0) * kChunk + (int64_t)threadIdx.x * 8;
  if (i >= t.n) return;
  double lr, lr1d, root2;
  corrections(a, &lr, &lr1d, &root2);
  const float b1 = (float)a.b1, b2 = (float)a.b2, omb1 = (float)a.omb1, omb2 = (float)a.omb2;
  const float eps = (float)a.eps, lrwd = (float)(lr * a.wd), lr1 = (float)lr1d;
  const float root = (float)root2;
  float p[8], g[8], m[8], v[8];
  float* mp = static_cast<float*>(a.m) + t.state0;
  float* vp = static_cast<float*>(a.v) + t.state0;
  get_typed(t.g, t.g_type, i, t.n, t.g_vec, g);
  get_typed(t.p, t.p_type, i, t.n, t.p_vec, p);
  get8(mp, i, t.n, true, m);
  get8(vp, i, t.n, true, v);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const float gq = g[q] * a.grad_scale;
    m[q] = fmaf(b1, m[q], omb1 * gq);
    v[q] = fmaf(b2, v[q], omb2 * gq * gq);
    const float den = fmaf(__builtin_sqrtf(v[q]), root, eps);
    p[q] = fmaf(-lrwd, p[q], p[q]) - m[q] * lr1 / den;
  }
  put8(mp, i, t.n, true, m);
  put8(vp, i, t.n, true, v);
  put_typed(t.p, t.p_type, i, t.n, t.p_vec, p);
}

// -- 8-bit codes -----------------------------------------------------------------------------------
// An unsigned float code of MANT mantissa bits stands for the integer
//     (e ? 2^MANT + f : f) << max(e - 1, 0),   e = c >> MANT, f = c & (2^MANT - 1),
// which is the float32 with the code's bits at the top of its exponent and mantissa fields, times
// 2^(126 + MANT): float32's own subnormals stand for the code's.
template <int MANT>
__device__ __forceinline__ float code_float(unsigned c) {
  return __uint_as_float(c << (23 - MANT));
}
// that factor, as a power of two for float64
constexpr double kMUnit = 0x1p129, kRUnit = 0x1p130;

// The code nearest to q >= 0 (in units of the smallest code above zero), a middle to the even one, at
// most `top`.  float64 bits: the exponent and the 20 mantissa bits of the upper word, the rest folded
// into a sticky bit, so that "exactly the middle" is told from "a little above it".  Below 2^MANT, where
// the grid is 1, q + 2^MANT has the same grid and 2^MANT codes more.
template <int MANT>
__device__ __forceinline__ unsigned nearest_code(double q, unsigned top) {
  const bool small = q < (double)(1 << MANT);
  const unsigned long long bits = __double_as_longlong(q + (small ? (double)(1 << MANT) : 0.0));
  unsigned hi = (unsigned)(bits >> 32);
  hi |= (unsigned)((unsigned)bits != 0u);            // sticky
  constexpr int kDrop = 20 - MANT;
  const unsigned r = hi + ((1u << (kDrop - 1)) - 1u) + ((hi >> kDrop) & 1u);
  // r >> kDrop = biased exponent and MANT bits; exponent MANT is code exponent 1
  const unsigned c = (r >> kDrop) - (((1023u + MANT - 1u) << MANT) + (small ? 1u << MANT : 0u));
  return c < top ? c : top;
}

// sqrt of a normal float64 > 0 to within its last bit or two: the hardware's estimate of 1 / sqrt and
// two steps of Newton's method (the library's also scales the exponent and handles every special value)
__device__ __forceinline__ double root_of(double v) {
  const double y = __builtin_amdgcn_rsq(v);
  double g = v * y, h = 0.5 * y;
  const double r = fma(-g, h, 0.5);
  g = fma(g, r, g);
  h = fma(h, r, h);
  return fma(fma(-g, g, v), h, g);
}
// 1 / x of a normal float64 to within its last bit or two, the same way
__device__ __forceinline__ double inverse_of(double x) {
  double y = __builtin_amdgcn_rcp(x);
  y = fma(fma(-x, y, 1.0), y, y);
  return fma(fma(-x, y, 1.0), y, y);
}
// v = 0 becomes kTiny, whose root is far below every scale; any v above zero has a larger root
constexpr double kTiny = 1e-290, kSeen = 1.1e-145;

// Largest over the 32 lanes that hold one block of 256 elements; values >= 0.
template <int CTRL>
__device__ __forceinline__ double dpp_max(double v) {
  const unsigned long long b = __double_as_longlong(v);
  const unsigned long long o = ((unsigned long long)dpp_u32<CTRL>(0u, (unsigned)(b >> 32)) << 32) |
                               dpp_u32<CTRL>(0u, (unsigned)b);
  return fmax(v, __longlong_as_double(o));
}
__device__ __forceinline__ double half_wave_max(double v) {
  v = dpp_max<0x111>(v);
  v = dpp_max<0x112>(v);
  v = dpp_max<0x114>(v);
  v = dpp_max<0x118>(v);
  v = dpp_max<0x142>(v);   // lane 31 now holds the first 32 lanes' value, lane 63 the others'
  const unsigned long long b = __double_as_longlong(v);
  const int lo = (int)(unsigned)b, hi = (int)(b >> 32);
  const bool first = (threadIdx.x & 32) == 0;
  const unsigned l = (unsigned)(first ? __builtin_amdgcn_readlane(lo, 31) : __builtin_amdgcn_readlane(lo, 63));
  const unsigned h = (unsigned)(first ? __builtin_amdgcn_readlane(hi, 31) : __builtin_amdgcn_readlane(hi, 63));
  return __longlong_as_double(((unsigned long long)h << 32) | l);
}
// |v|, or next to nothing where v is not finite
__device__ __forceinline__ double finite_size(double v) {
  const unsigned long long b = __double_as_longlong(v) & 0x7fffffffffffffffull;
  const unsigned hi = (unsigned)(b >> 32);
  const unsigned keep = hi < 0x7ff00000u ? hi : 0u;
  return __longlong_as_double(((unsigned long long)keep << 32) | (unsigned)b);
}

// What a lane needs besides its elements: the block's old scales as the codes' units, the step.
struct Lane8 {
  double sm, sv;      // times a code's float32 (code_float) = the value
  double b1, b2, omb1, omb2, root;
  float lr1, lrwd, eps;
};

// WIDE: for divisors up to the largest float32.  The hardware's reciprocal flushes what is below 2^-126, so a quarter
// of the divisor is inverted (none of a float32 has so small a reciprocal, none of an eps from 2^-124 on too large a one).
template <bool WIDE>
__device__ __forceinline__ float stepped(float p, float m, double r, const Lane8& s) {
  if (!WIDE) return fmaf(-s.lrwd, p, p) - m * s.lr1 * __builtin_amdgcn_rcpf((float)(r * s.root) + s.eps);
  const float quarter = 0.25f * __builtin_amdgcn_rcpf((float)(0.25 * (r * s.root)) + 0.25f * s.eps);
  return fmaf(-s.lrwd, p, p) - m * s.lr1 * quarter;
}

// A block of 256 elements is held by 32 lanes, eight elements each, from the codes to the new codes.
//
// adamw8_careful decides every code in float64 and handles what is not finite.
// adamw8_quick is for finite values.  Its codes come from the float64 quotients rounded to float32
// once: m's by the hardware's conversion to this format (e4m3), v's from the float32 bits.  That is the
// same code except in two cases: where the float32 is exactly a middle between two codes (one in 2^19 or so), and
// where a new scale is a float32 subnormal.  Rounding such a scale moves it by up to a half, so the largest quotient
// may pass the largest code, and neither of these codes is bounded (e4m3 has no number above 464, v's bits run into
// the next byte); a normal scale moves by 2^-24 at most, which float32 quotients do not see.  In both, and where a
// divisor of the step is above 2^122 (stepped), it returns true and the wave takes the careful way instead.
__device__ __forceinline__ void adamw8_careful(const Lane8& s, u32x2 mc, u32x2 vc, const float* g, const float* p,
                                               float* p_out, u32x2* mo, u32x2* vo, float* out_sm, float* out_sv) {
  double m[8], r[8];
  double top_m = 0.0, top_r = 0.0;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const double gq = (double)g[q];
    const unsigned cm = (mc[q >> 2] >> (8 * (q & 3))) & 255u, cv = (vc[q >> 2] >> (8 * (q & 3))) & 255u;
    float fm = __uint_as_float(__float_as_uint(code_float<3>(cm & 127u)) | ((cm & 128u) << 24));
    float fr = code_float<4>(cv);
    fm = (cm & 127u) == 127u ? __builtin_nanf("") : fm;
    fr = cv == 255u ? __builtin_nanf("") : fr;
    const double r0 = (double)fr * s.sv;
    m[q] = fma(s.b1, (double)fm * s.sm, s.omb1 * gq);
    const double v = fma(s.b2, r0 * r0, s.omb2 * (gq * gq));
    r[q] = root_of(v > kTiny ? v : v + kTiny);   // (NaN stays)
    p_out[q] = stepped<true>(p[q], (float)m[q], r[q], s);
    top_m = fmax(top_m, finite_size(m[q]));
    top_r = fmax(top_r, finite_size(r[q]));
  }
  const float new_sm = (float)(half_wave_max(top_m) * (1.0 / 448.0));
  const float new_sv = (float)(half_wave_max(top_r) * (1.0 / 491520.0));
  const double im = new_sm > 0.0f ? 512.0 * inverse_of((double)new_sm) : 0.0;
  const double iv = new_sv > 0.0f ? inverse_of((double)new_sv) : 0.0;
  const double seen = new_sv > 0.0f ? kSeen : __builtin_inf();
  *mo = u32x2{0u, 0u};
  *vo = u32x2{0u, 0u};
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    unsigned cm = nearest_code<3>(fabs(m[q]) * im, 126u);
    unsigned cv = nearest_code<4>(r[q] * iv, 254u);
    const unsigned least = r[q] > seen ? 1u : 0u;
    cv = cv > least ? cv : least;
    cm = fabs(m[q]) < __builtin_inf() ? cm : 127u;
    cv = r[q] < __builtin_inf() ? cv : 255u;
    cm |= m[q] < 0.0 ? 128u : 0u;
    (*mo)[q >> 2] |= cm << (8 * (q & 3));
    (*vo)[q >> 2] |= cv << (8 * (q & 3));
  }
  *out_sm = new_sm;
  *out_sv = new_sv;
}

__device__ __forceinline__ bool adamw8_quick(const Lane8& s, u32x2 mc, u32x2 vc, const float* g, const float* p,
                                             float* p_out, u32x2* mo, u32x2* vo, float* out_sm, float* out_sv) {
  double m[8], r[8];
  double top_m = 0.0, top_r = 0.0;
  // (the hardware decodes m in units of the scale; code_float's unit is 2^-129 of it)
  const double b1sm = s.b1 * s.sm * 0x1p-120, b2sv2 = s.b2 * (s.sv * s.sv);
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    const double gq = (double)g[q];
    const int w = (int)mc[q >> 2];
    const float fm = (q & 3) == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0)
                     : (q & 3) == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1)
                     : (q & 3) == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2)
                                    : __builtin_amdgcn_cvt_f32_fp8(w, 3);
    const double fr = (double)code_float<4>((vc[q >> 2] >> (8 * (q & 3))) & 255u);
    m[q] = fma((double)fm, b1sm, s.omb1 * gq);
    const double v = fma(fr * fr, b2sv2, s.omb2 * (gq * gq));
    r[q] = root_of(fmax(v, kTiny));
    p_out[q] = stepped<false>(p[q], (float)m[q], r[q], s);
    top_m = fmax(top_m, fabs(m[q]));
    top_r = fmax(top_r, r[q]);
  }
  const float new_sm = (float)(half_wave_max(top_m) * (1.0 / 448.0));
  const float new_sv = (float)(half_wave_max(top_r) * (1.0 / 491520.0));
  const double im = new_sm > 0.0f ? inverse_of((double)new_sm) : 0.0;
  const double iv = new_sv > 0.0f ? inverse_of((double)new_sv) : 0.0;
  const double seen = new_sv > 0.0f ? kSeen : __builtin_inf();
  bool doubt = (new_sm > 0.0f && new_sm < 0x1p-126f) || (new_sv > 0.0f && new_sv < 0x1p-126f) ||
               new_sv * (491520.0f * (float)s.root) > 0x1p122f;
  float qm[8];
  *vo = u32x2{0u, 0u};
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    qm[q] = (float)(m[q] * im);
    // below 2^-6 e4m3's grid is that of [2^-6, 2^-5)
    const float am = fabsf(qm[q]);
    const float t = am + (am < 0x1p-6f ? 0x1p-6f : 0.0f);
    doubt |= (__float_as_uint(t) & 0xfffffu) == 0x80000u;
    // v: below 16 the grid is that of [16, 32)
    float qv = (float)(r[q] * iv);
    qv = r[q] > seen ? fmaxf(qv, 1.0f) : 0.0f;
    const bool small = qv < 16.0f;
    const unsigned bits = __float_as_uint(qv + (small ? 16.0f : 0.0f));
    doubt |= (bits & 0x7ffffu) == 0x40000u;
    // exponent 4 is code exponent 1
    const unsigned base = small ? (131u << 23) : (130u << 23);
    const unsigned cv = (bits + 0x3ffffu + ((bits >> 19) & 1u) - base) >> 19;
    (*vo)[q >> 2] |= cv << (8 * (q & 3));
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    int c = __builtin_amdgcn_cvt_pk_fp8_f32(qm[4 * w], qm[4 * w + 1], 0, false);
    c = __builtin_amdgcn_cvt_pk_fp8_f32(qm[4 * w + 2], qm[4 * w + 3], c, true);
    (*mo)[w] = (unsigned)c;
  }
  *out_sm = new_sm;
  *out_sv = new_sv;
  return doubt;
}

// 32 lanes share a block of states, 8 elements each.  128 Mi bf16 parameters in 40 tensors: 430 to 510 us,
// 2.6 to 3.1 TB/s: bound by its vector instructions (memory alone is 260 us; with every code decided in
// float64 589 us, with states decoded by exponent arithmetic 699).
__global__ __launch_bounds__(256) void k_adamw8(AdamTable tab, AdamArgs a) {
  const int chunk = blockIdx.x;
  const AdamTensor& t = tab.t[find_tensor(tab, chunk)];
  const int64_t i = (int64_t)(chunk - t.chunk0) * kChunk + (int64_t)threadIdx.x * 8;
  const int64_t padded = (t.n + kStateBlock - 1) / kStateBlock * kStateBlock;
  if (i >= padded) return;   // whole blocks: their 32 lanes stay together
  double lr, lr1d, root;
  corrections(a, &lr, &lr1d, &root);
  // (the step itself is float32: only what becomes a code has to be decided in float64)
  // (an eps whose reciprocal is no float32 would turn a step of 0 / eps into NaN)
  const float lr1 = (float)lr1d, lrwd = (float)(lr * a.wd), eps = fmaxf((float)a.eps, 0x1p-124f);
  unsigned char* mp = static_cast<unsigned char*>(a.m) + t.state0 + i;
  unsigned char* vp = static_cast<unsigned char*>(a.v) + t.state0 + i;
  const int64_t block = (t.state0 + i) / kStateBlock;
  u32x2 mc = *reinterpret_cast<const u32x2*>(mp);
  u32x2 vc = *reinterpret_cast<const u32x2*>(vp);
  const double sm = (double)a.scale_m[block] * (kMUnit / 512.0), sv = (double)a.scale_v[block] * kRUnit;
  float p[8], g[8];
  get_typed(t.g, t.g_type, i, t.n, t.g_vec, g);
  get_typed(t.p, t.p_type, i, t.n, t.p_vec, p);
  if (i + 8 > t.n) {   // behind the tensor's end the states are 0, and so are p and g (get8)
#pragma unroll
    for (int q = 0; q < 8; ++q)
      if (i + q >= t.n) {
        mc[q >> 2] &= ~(255u << (8 * (q & 3)));
        vc[q >> 2] &= ~(255u << (8 * (q & 3)));
      }
  }
  // anything that is not finite: x * 0 is NaN then; a byte of m with all of its lower seven bits set, or
  // of v with all eight
  float odd = 0.0f;
#pragma unroll
  for (int q = 0; q < 8; ++q) {
    g[q] *= a.grad_scale;
    odd = fmaf(g[q], 0.0f, odd);
  }
  unsigned marks = 0;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    marks |= ((mc[w] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    marks |= ((vc[w] & 0x7f7f7f7fu) + 0x01010101u) & vc[w] & 0x80808080u;
  }
  const Lane8 l{sm, sv, a.b1, a.b2, a.omb1, a.omb2, root, lr1, lrwd, eps};
  u32x2 mo, vo;
  float p_out[8], new_sm, new_sv;
  bool again = marks != 0u || odd != odd;
  if (!__ballot(again)) again = adamw8_quick(l, mc, vc, g, p, p_out, &mo, &vo, &new_sm, &new_sv);
  if (__ballot(again)) adamw8_careful(l, mc, vc, g, p, p_out, &mo, &vo, &new_sm, &new_sv);
  put_typed(t.p, t.p_type, i, t.n, t.p_vec, p_out);
  *reinterpret_cast<u32x2*>(mp) = mo;
  *reinterpret_cast<u32x2*>(vp) = vo;
  if ((threadIdx.x & 31) == 0) {
    a.scale_m[block] = new_sm;
    a.scale_v[block] = new_sv;
  }
}

// The float32 values that 8-bit states stand for.  128 Mi of either: 215 us, 6.2 TB/s: bound by memory.
__global__ __launch_bounds__(256) void k_adamw_values(const unsigned char* mc, const unsigned char* vc,
                                                      const float* scale_m, const float* scale_v,
                                                      int64_t n, float* m, float* v) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= n) return;
  const unsigned cm = *reinterpret_cast<const unsigned*>(mc + i);
  const unsigned cv = *reinterpret_cast<const unsigned*>(vc + i);
  const float sm = scale_m[i / kStateBlock], sv = scale_v[i / kStateBlock];
  f32x4 om, ov;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const unsigned c = (cm >> (8 * q)) & 255u, d = (cv >> (8 * q)) & 255u;
    const float x = (float)((double)code_float<3>(c & 127u) * (kMUnit / 512.0)) * sm;
    om[q] = (c & 127u) == 127u ? __builtin_nanf("") : (c & 128u) ? -x : x;
    const float y = (float)((double)code_float<4>(d) * kRUnit) * sv;
    ov[q] = d == 255u ? __builtin_nanf("") : y * y;
  }
  *reinterpret_cast<f32x4*>(m + i) = om;
  *reinterpret_cast<f32x4*>(v + i) = ov;
}

}  // namespace

hipError_t launch_adamw(const AdamTensor* tensors, int64_t count, int bits, void* m, void* v,
                        float* scales, int64_t state_elements, double lr, const float* lr_dev,
                        double b1, double b2, double eps, double wd, int64_t step,
                        const int64_t* step_dev, float grad_scale, hipStream_t s) {
  AdamArgs a;
  a.m = m;
  a.v = v;
  a.scale_m = scales;
  a.scale_v = scales ? scales + state_elements / kStateBlock : nullptr;
  a.lr = lr;
  a.b1 = b1;
  a.b2 = b2;
  a.omb1 = 1.0 - b1;
  a.omb2 = 1.0 - b2;
  a.eps = eps;
  a.wd = wd;
  double p1 = 1.0, p2 = 1.0;
  double q1 = b1, q2 = b2;
  for (int64_t t = step; t > 0; t >>= 1) {
    if (t & 1) {
      p1 *= q1;
      p2 *= q2;
    }
    q1 *= q1;
    q2 *= q2;
  }
  a.c1 = 1.0 - p1;
  a.c2 = 1.0 - p2;
  a.lr1 = lr / a.c1;
  a.root2 = std::sqrt(1.0 / a.c2);
  a.lr_dev = lr_dev;
  a.step_dev = step_dev;
  a.grad_scale = grad_scale;
  AdamTable tab;
  int64_t i = 0;
  while (i < count) {
    tab.count = 0;
    int64_t chunks = 0;
    for (; i < count && tab.count < kTensorsPerLaunch; ++i) {
      if (tensors[i].n == 0) continue;
      const int64_t more = (tensors[i].n + kChunk - 1) / kChunk;
      if (chunks + more > kMaxChunks) {
        if (tab.count) break;              // the next launch begins with it
        return hipErrorInvalidValue;       // (refused by the caller's checks)
      }
      AdamTensor& d = tab.t[tab.count++];
      d = tensors[i];
      d.chunk0 = (int)chunks;
      d.p_vec = (reinterpret_cast<uintptr_t>(d.p) & 15) == 0;
      d.g_vec = (reinterpret_cast<uintptr_t>(d.g) & 15) == 0;
      chunks += more;
    }
    if (!tab.count) break;
    if (bits == 8) hipLaunchKernelGGL(k_adamw8, dim3((unsigned)chunks), dim3(256), 0, s, tab, a);
    else hipLaunchKernelGGL(k_adamw32, dim3((unsigned)chunks), dim3(256), 0, s, tab, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_adamw_values(const unsigned char* m, const unsigned char* v, const float* scales,
                               int64_t n, float* out_m, float* out_v, hipStream_t s) {
  const int64_t per = (int64_t)1 << 32;   // elements of a launch (a multiple of kStateBlock)
  for (int64_t i = 0; i < n; i += per) {
    const int64_t k = n - i < per ? n - i : per;
    hipLaunchKernelGGL(k_adamw_values, dim3((unsigned)((k + 1023) / 1024)), dim3(256), 0, s, m + i,
                       v + i, scales + i / kStateBlock, scales + (n + i) / kStateBlock, k, out_m + i,
                       out_v + i);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace ic
