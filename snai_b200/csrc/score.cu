// score.cu - operators over rows of vocabulary logits: log probabilities of
// given tokens with entropy and top alternatives, their gradient, and the
// distillation loss against a teacher's top logits with its gradient
// (cortex_score, cortex_score_grad, cortex_distill in include/cortex.h).
//
// With T the temperature, m the row's maximum, d_i = (z_i - m) / T,
// e_i = exp(d_i) and S = sum e_i:
//   log p_i = d_i - log S,  entropy H = log S - sum(e_i d_i) / S.
// A masked logit (-inf) has e_i = 0 and takes no gradient; a row holding a
// NaN or +inf has no distribution: its S is NaN and so is all that follows
// (its alternatives' ids -1).
//
// All three read a row once from memory and are bound by that (and by the
// gradient's one write).  16-byte words are copied to shared memory
// asynchronously, each by the thread that will read it, so no barrier stands
// between a copy and its use.  Pass A takes four words at a time (a chunk) and
// gathers the reference m, S and sum(e d) together.  Scores need no more and
// stream through a ring; a gradient needs the row again, which stays staged,
// cut into slices over a cluster of CTAs when it is long.
//
// Measured on a B200 against its copy rate of 6553 GB/s (the bytes each
// operator cannot do without over its time): 2048 x 131072 fp32 scores 1.05,
// with 64 alternatives 0.70, distillation with the rest 0.87; 8192 x 16384
// fp32 scores with 20 alternatives 0.57, gradient 0.83, distillation of 64
// entries with labels 0.86; 8192 x 32000 bf16 scores 0.81 and 2048 x 131072
// bf16 gradient 0.78, where two bytes an element bring 9 and 15 lane
// instructions: 70 and 56 % of the issue slots, 64 and 60 % of the pipe of
// exponentials and conversions, none full, waiting for one another.
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cmath>
#include <exception>
#include <initializer_list>
#include <map>
#include <mutex>
#include <tuple>
#include <utility>

#include "../../include/cortex.h"
#include "common.cuh"
#include "engine.h"

namespace snai {
namespace {

constexpr int kMaxList = kScoreMaxK;
constexpr int kMaxVocab = 1 << 19;  // as cortex_sample
constexpr int kMaxRows = 1 << 30;
constexpr long long kMaxElems = 1ll << 48;  // rows x stride: byte offsets stay far inside 64 bits
constexpr int kStages = 4;          // copy groups a row's words are committed in
constexpr int kChunk = 4;           // words a thread takes at a time
constexpr float kLowest = -200.f;   // exponents (base 2) are cut here: 2^-200 is 0 in fp32, and 0 * d stays 0
constexpr double kLn2d = 0.69314718055994531;
constexpr float kLn2 = 0.69314718055994531f, kLog2E = 1.4426950408889634f;

// ---- small device pieces ----

// maxima that keep a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
  float r;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}
// The hardware's 2^x is low by this in the mean below x = -1 (measured: 2^20
// arguments in each of four ranges down to -60 gave 4.98 to 5.16e-8; exact at
// 0, at most 1.5e-7 off): a sum of many such terms is, and a distillation loss,
// a small difference of such sums' logarithms, takes it out (1024 rows of
// 16384, mean error of losses of 1e-3: 2e-8 without, 2e-9 with it).  For a row
// of a few terms it is not their own error, but less than a step of fp32.
// Scores and the label's loss are rounded to fp32 at their own size and keep it.
constexpr double kEx2Low = 5e-8;
__device__ __forceinline__ float ex2(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// two floats in a register pair
typedef unsigned long long f2;
__device__ __forceinline__ f2 pack2(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(f2 v, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sum2(f2 v) {
  float a, b;
  unpack2(v, a, b);
  return a + b;
}

// Eight bits, in order, from four pairs of 16-bit masks.
__device__ __forceinline__ unsigned reach8(unsigned a, unsigned b, unsigned c, unsigned d) {
  // pair i's low half gives bit 2 i, its high half bit 16 + 2 i + 1
  const unsigned v = (a & 0x00020001u) | (b & 0x00080004u) | (c & 0x00200010u) | (d & 0x00800040u);
  return (v | v >> 16) & 0xffu;
}

// A 16-byte word of logits: kN elements; kMasked is -inf in each of its 32-bit parts.
template <typename E> struct Word;
template <> struct Word<float> {
  static constexpr int kN = 4;
  static constexpr unsigned kMasked = 0xff800000u;
  __device__ static __forceinline__ void unpack(const uint4 &w, f2 *v) {
    v[0] = pack2(__uint_as_float(w.x), __uint_as_float(w.y));
    v[1] = pack2(__uint_as_float(w.z), __uint_as_float(w.w));
  }
  __device__ static __forceinline__ uint4 pack(const f2 *v) {
    float a, b, c, d;
    unpack2(v[0], a, b);
    unpack2(v[1], c, d);
    return make_uint4(__float_as_uint(a), __float_as_uint(b), __float_as_uint(c), __float_as_uint(d));
  }
  // maximum over N words
  template <int N> __device__ static __forceinline__ float max(const uint4 *q) {
    float m = __uint_as_float(q[0].x);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      m = max_nan(m, max_nan(__uint_as_float(q[j].x), __uint_as_float(q[j].y)));
      m = max_nan(m, max_nan(__uint_as_float(q[j].z), __uint_as_float(q[j].w)));
    }
    return m;
  }
  // one bit for each element that reaches limit(least)
  __device__ static __forceinline__ unsigned limit(float least) { return __float_as_uint(least); }
  __device__ static __forceinline__ unsigned reach(const uint4 &w, unsigned lim) {
    const float l = __uint_as_float(lim);
    return (__uint_as_float(w.x) >= l ? 1u : 0u) | (__uint_as_float(w.y) >= l ? 2u : 0u) |
           (__uint_as_float(w.z) >= l ? 4u : 0u) | (__uint_as_float(w.w) >= l ? 8u : 0u);
  }
  __device__ static __forceinline__ float one(const float *p) { return *p; }
  __device__ static __forceinline__ void put(float *p, float v) { *p = v; }
};
template <> struct Word<__nv_bfloat16> {
  static constexpr int kN = 8;
  static constexpr unsigned kMasked = 0xff80ff80u;
  __device__ static __forceinline__ f2 two(unsigned x) {
    return pack2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  }
  __device__ static __forceinline__ unsigned two(f2 v) {
    float a, b;
    unpack2(v, a, b);
    unsigned r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  __device__ static __forceinline__ void unpack(const uint4 &w, f2 *v) {
    v[0] = two(w.x), v[1] = two(w.y), v[2] = two(w.z), v[3] = two(w.w);
  }
  __device__ static __forceinline__ uint4 pack(const f2 *v) {
    return make_uint4(two(v[0]), two(v[1]), two(v[2]), two(v[3]));
  }
  __device__ static __forceinline__ unsigned max2(unsigned a, unsigned b) {
    unsigned r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  template <int N> __device__ static __forceinline__ float max(const uint4 *q) {
    unsigned m = q[0].x;
#pragma unroll
    for (int j = 0; j < N; ++j) m = max2(m, max2(max2(q[j].x, q[j].y), max2(q[j].z, q[j].w)));
    return max_nan(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  __device__ static __forceinline__ unsigned limit(float least) {
    const __nv_bfloat162 v = __bfloat162bfloat162(__float2bfloat16_ru(least));
    return *reinterpret_cast<const unsigned *>(&v);
  }
  __device__ static __forceinline__ unsigned ge2(unsigned a, unsigned lim) {
    return __hge2_mask(*reinterpret_cast<const __nv_bfloat162 *>(&a), *reinterpret_cast<const __nv_bfloat162 *>(&lim));
  }
  __device__ static __forceinline__ unsigned reach(const uint4 &w, unsigned lim) {
    return reach8(ge2(w.x, lim), ge2(w.y, lim), ge2(w.z, lim), ge2(w.w, lim));
  }
  __device__ static __forceinline__ float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
  __device__ static __forceinline__ void put(__nv_bfloat16 *p, float v) { *p = __float2bfloat16_rn(v); }
};
template <> struct Word<__half> {
  static constexpr int kN = 8;
  static constexpr unsigned kMasked = 0xfc00fc00u;
  __device__ static __forceinline__ f2 two(unsigned x) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&x));
    return pack2(f.x, f.y);
  }
  __device__ static __forceinline__ unsigned two(f2 v) {
    float a, b;
    unpack2(v, a, b);
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
  }
  __device__ static __forceinline__ void unpack(const uint4 &w, f2 *v) {
    v[0] = two(w.x), v[1] = two(w.y), v[2] = two(w.z), v[3] = two(w.w);
  }
  __device__ static __forceinline__ uint4 pack(const f2 *v) {
    return make_uint4(two(v[0]), two(v[1]), two(v[2]), two(v[3]));
  }
  __device__ static __forceinline__ unsigned max2(unsigned a, unsigned b) {
    unsigned r;
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  template <int N> __device__ static __forceinline__ float max(const uint4 *q) {
    unsigned m = q[0].x;
#pragma unroll
    for (int j = 0; j < N; ++j) m = max2(m, max2(max2(q[j].x, q[j].y), max2(q[j].z, q[j].w)));
    float a, b;
    unpack2(two(m), a, b);
    return max_nan(a, b);
  }
  __device__ static __forceinline__ unsigned limit(float least) {
    const __half2 v = __half2half2(__float2half_ru(least));
    return *reinterpret_cast<const unsigned *>(&v);
  }
  __device__ static __forceinline__ unsigned ge2(unsigned a, unsigned lim) {
    return __hge2_mask(*reinterpret_cast<const __half2 *>(&a), *reinterpret_cast<const __half2 *>(&lim));
  }
  __device__ static __forceinline__ unsigned reach(const uint4 &w, unsigned lim) {
    return reach8(ge2(w.x, lim), ge2(w.y, lim), ge2(w.z, lim), ge2(w.w, lim));
  }
  __device__ static __forceinline__ float one(const __half *p) { return __half2float(*p); }
  __device__ static __forceinline__ void put(__half *p, float v) { *p = __float2half_rn(v); }
};

// Sort key of a logit and its id: descending value, then ascending id.
__device__ __forceinline__ unsigned long long sort_key(float z, int id) {
  const int b = __float_as_int(z + 0.0f);  // -0 counts as +0
  const unsigned k = (unsigned)b ^ (b < 0 ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)k << 32) | (unsigned)~id;
}
__device__ __forceinline__ float key_logit(unsigned long long key) {
  const unsigned k = (unsigned)(key >> 32);
  return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int key_id(unsigned long long key) { return (int)~(unsigned)key; }

// ---- rows in shared memory ----

struct Rows {
  const void *logits;
  long long ld;
  int rows, V;
  int wps;    // words of a slice
  int C;      // CTAs of a cluster, one slice each
  bool even;  // all rows start at the same place of a 16-byte word
};

// The word at p whose element 0 is id0 of a row of V, -inf beyond the row's
// ends; and such a word's elements to the row at out.  By value, and not
// members: an object whose address a call takes lives in local memory.
template <typename E>
__device__ __noinline__ uint4 ragged(const char *p, int id0, int V) {
  __align__(16) E v[Word<E>::kN];
#pragma unroll
  for (int k = 0; k < Word<E>::kN; ++k)
    Word<E>::put(v + k,
                 id0 + k >= 0 && id0 + k < V ? Word<E>::one(reinterpret_cast<const E *>(p) + k) : -INFINITY);
  return *reinterpret_cast<const uint4 *>(v);
}
template <typename E>
__device__ __noinline__ void put_ragged(uint4 q, E *out, int id0, int V) {
  const E *v = reinterpret_cast<const E *>(&q);
#pragma unroll
  for (int k = 0; k < Word<E>::kN; ++k)
    if (id0 + k >= 0 && id0 + k < V) out[id0 + k] = v[k];
}

// One CTA's slice of one row: words [first, first + n) of the row's 16-byte
// grid, which starts `pad` elements before the row when the row does not
// start on a word.  Thread t owns words t, t + NT, ... of the slice.  All
// words are whole but the row's first and last, when they are ragged: whole
// words are [lo, hi).
template <typename E, int NT>
struct Slice {
  static constexpr int kN = Word<E>::kN;
  static constexpr int kWide = kChunk * NT;  // words of a chunk over all threads
  const char *src;  // the slice's word 0
  int base;         // id of its element 0 (negative in the leading pad)
  int n, lo, hi, V;

  __device__ __forceinline__ void set(const Rows &a, int r, unsigned rank) {
    const char *row = static_cast<const char *>(a.logits) + (long long)r * a.ld * (int)sizeof(E);
    const int pad = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(E));
    const int first = (int)rank * a.wps, words = (pad + a.V + kN - 1) / kN;
    V = a.V;
    base = first * kN - pad;
    src = row + (long long)base * (int)sizeof(E);
    n = min(a.wps, words - first);
    lo = base < 0 ? 1 : 0;
    hi = base + n * kN > V ? n - 1 : n;
  }
  // the slice of row r + step
  __device__ __forceinline__ void next(const Rows &a, int r, int step, unsigned rank) {
    if (a.even)
      src += (long long)step * a.ld * (int)sizeof(E);
    else
      set(a, r + step, rank);
  }
  __device__ __forceinline__ int id0(int w) const { return base + w * kN; }
  // local element index of an id, negative when another slice holds it
  __device__ __forceinline__ int local(int id) const {
    const int e = id - base;
    return e < n * kN ? e : -1;
  }
  __device__ __forceinline__ const E *at(int id) const {
    return reinterpret_cast<const E *>(src + (long long)(id - base) * (int)sizeof(E));
  }
  // Copies this thread's words of chunk c to `to` (a chunk's place in shared
  // memory).  The row's ragged ends are filled up with -inf.
  __device__ __forceinline__ void load_chunk(int c, uint4 *to) const {
    const int w0 = c * kWide;
    const uint32_t dst = smem_u32(to + threadIdx.x);
    const char *p = src + (long long)(w0 + (int)threadIdx.x) * 16;
    if (w0 >= lo && w0 + kWide <= hi) {
#pragma unroll
      for (int j = 0; j < kChunk; ++j) copy16(dst + j * NT * 16, p + j * NT * 16);
    } else {
#pragma unroll
      for (int j = 0; j < kChunk; ++j) {
        const int w = w0 + j * NT + (int)threadIdx.x;
        if (w >= lo && w < hi)
          copy16(dst + j * NT * 16, p + j * NT * 16);
        else if (w < n)
          to[w - w0] = ragged<E>(p + j * NT * 16, id0(w), V);
      }
    }
  }
  // the words of stage st (cps chunks) of a row staged as a whole, committed as one group
  __device__ __forceinline__ void load(int st, int cps, uint4 *buf) const {
    for (int c = st * cps; c < (st + 1) * cps && c * kWide < n; ++c) load_chunk(c, buf + c * kWide);
    commit();
  }
  __device__ static __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  __device__ static __forceinline__ void copy16(uint32_t dst, const char *p) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(p) : "memory");
  }
  // word w from global memory, masked beyond the row's ends
  __device__ __forceinline__ uint4 fetch(int w) const {
    const char *p = src + (long long)w * 16;
    if (w >= lo && w < hi) return *reinterpret_cast<const uint4 *>(p);
    return ragged<E>(p, id0(w), V);
  }
  // stores word w of a row whose element 0 is at out
  __device__ __forceinline__ void store_ragged(int w, const uint4 &q, E *out) const {
    put_ragged(q, out, id0(w), V);
  }
  // this thread's four words of chunk c, staged at `at` (all masked past the slice's end)
  __device__ __forceinline__ void chunk(int c, const uint4 *at, uint4 *q) const {
    at += threadIdx.x;
    if ((c + 1) * kWide <= n) {
#pragma unroll
      for (int j = 0; j < kChunk; ++j) q[j] = at[j * NT];
    } else {
      constexpr unsigned k = Word<E>::kMasked;
      const int left = n - c * kWide - (int)threadIdx.x;
#pragma unroll
      for (int j = 0; j < kChunk; ++j) q[j] = j * NT < left ? at[j * NT] : make_uint4(k, k, k, k);
    }
  }
};

template <int N> __device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void copies_wait(int n) {  // n < kStages
  if (n == 0)
    copies_wait<0>();
  else if (n == 1)
    copies_wait<1>();
  else if (n == 2)
    copies_wait<2>();
  else
    copies_wait<3>();
}

// ---- softmax statistics ----

// m, S = sum 2^((z - m) c) and, when asked, W = sum 2^x x (x = (z - m) c) and
// S1 = sum 2^((z - m) log2 e), the sum at temperature 1.  All masked: m is
// the lowest float and S 0.  A NaN or +inf makes S NaN.
struct Stat {
  float m, s, w, s1;
};
__device__ __forceinline__ float cut(float x) { return max_nan(x, kLowest); }

// a's sums relative to the maximum m >= a.m
template <bool W, bool S1>
__device__ __forceinline__ void rebase(Stat &a, float m, float c) {
  const float x = cut((a.m - m) * c), f = ex2(x);
  if (W) a.w = f * fmaf(a.s, x, a.w);
  a.s *= f;
  if (S1) a.s1 *= ex2(cut((a.m - m) * kLog2E));
  a.m = m;
}

// exp(d) from e = exp(d / T): its square or fourth power (SQ squarings), or by itself.
template <int SQ>
__device__ __forceinline__ f2 at_one(f2 e, f2 d, f2 l2) {
  if (SQ) {
    e = mul2(e, e);
    return SQ == 2 ? mul2(e, e) : e;
  }
  float a, b;
  unpack2(mul2(d, l2), a, b);
  return pack2(ex2(a), ex2(b));
}

// A thread's statistics as its words come.  m need not be the maximum: sums
// relative to a value up to 2^kAbove below it are as good (a sum of 2^19 terms
// stays far from fp32's end), so they are rebased only when a chunk's maximum
// cm passes that: once or twice a row instead of at most chunks.
constexpr float kAbove = 16.f;
template <typename E, bool W, bool S1, int SQ = 0>
struct Running {
  float m = -FLT_MAX, most = -FLT_MAX;
  f2 s = 0, w = 0, s1 = 0;

  __device__ __forceinline__ void add(const uint4 *q, float cm, float c, float above) {
    if (!(cm <= most)) {  // far above, or a NaN
      const float nm = max_nan(m, cm), x = cut((m - nm) * c), f = ex2(x);
      const f2 ff = pack2(f, f);
      if (W) w = mul2(ff, fma2(s, pack2(x, x), w));
      s = mul2(ff, s);
      if (S1) {
        const float f1 = ex2(cut((m - nm) * kLog2E));
        s1 = mul2(pack2(f1, f1), s1);
      }
      m = nm;
      most = nm + above;
    }
    // Without W a chunk's terms are summed by themselves: fewer roundings at the
    // sum's size, at no cost; with W the second set of sums costs 2 % (scores
    // of 8192 x 32000 bf16 99 us for 97).
    f2 cs = 0, cs1 = 0;
    const f2 nm2 = pack2(-m, -m), c2 = pack2(c, c), l2 = pack2(kLog2E, kLog2E);
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      f2 v[Word<E>::kN / 2];
      Word<E>::unpack(q[j], v);
#pragma unroll
      for (int k = 0; k < Word<E>::kN / 2; ++k) {
        const f2 d = add2(v[k], nm2);
        f2 x = mul2(d, c2);
        float a, b;
        unpack2(x, a, b);
        if (W) {
          a = cut(a), b = cut(b);
          x = pack2(a, b);
        }
        const f2 e = pack2(ex2(a), ex2(b));
        if (W) {
          s = add2(s, e);
          w = fma2(e, x, w);
          if (S1) s1 = add2(s1, at_one<SQ>(e, d, l2));
        } else {
          cs = j == 0 && k == 0 ? e : add2(cs, e);
          if (S1) cs1 = j == 0 && k == 0 ? at_one<SQ>(e, d, l2) : add2(cs1, at_one<SQ>(e, d, l2));
        }
      }
    }
    if (!W) s = add2(s, cs);
    if (!W && S1) s1 = add2(s1, cs1);
  }
  __device__ __forceinline__ Stat get() const { return {m, sum2(s), W ? sum2(w) : 0.f, S1 ? sum2(s1) : 0.f}; }
};

// Combines the statistics of n lanes (a power of two; lanes of equal number
// modulo n hold the same ones); every lane gets the result.
template <bool W, bool S1>
__device__ __forceinline__ Stat combine_lanes(Stat a, int n, float c) {
  rebase<W, S1>(a, warp_max_nan(a.m), c);
  for (int o = n / 2; o > 0; o >>= 1) {
    a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
    if (W) a.w += __shfl_xor_sync(0xffffffffu, a.w, o);
    if (S1) a.s1 += __shfl_xor_sync(0xffffffffu, a.s1, o);
  }
  return a;
}
__device__ __forceinline__ Stat no_stat() { return {-FLT_MAX, 0.f, 0.f, 0.f}; }

// What a CTA tells the others of its cluster about its slice.
struct __align__(16) Slip {
  Stat st;
  float tau;  // a bound of its alternatives (scores)
};

__device__ __forceinline__ Stat peer_stat(const Slip *mine, unsigned rank) {
  const uint32_t p = mapa_shared(smem_u32(mine), rank);
  return {__uint_as_float(ld_cluster_u32(p)), __uint_as_float(ld_cluster_u32(p + 4)),
          __uint_as_float(ld_cluster_u32(p + 8)), __uint_as_float(ld_cluster_u32(p + 12))};
}

// ---- scores ----

struct ScoreArgs {
  Rows in;
  const int *tokens;
  int n_tok;
  float c;               // log2(e) / T, rounded
  float two_t, two_t_lo;  // 2 / T in two parts
  float off;             // what c's rounding takes from log S, over W / S
  int top_k, cap, soft, grow;  // candidates: what the buffer holds (a power of two), where it is thinned out, and when
  float *logprob, *entropy;
  int *top_ids;
  float *top_logprob;
};

// log p of a logit; ls is log S.  Half the difference never passes fp32's
// range, where the difference of logits at both of its ends would: over T it
// may be back inside.
__device__ __forceinline__ float log_p(const ScoreArgs &a, float z, float m, float s, float ls) {
  const float d = fmaf(0.5f, z, -0.5f * m);
  return s == 0.f || z == -INFINITY ? -INFINITY + (s - s) : fmaf(d, a.two_t, fmaf(d, a.two_t_lo, -ls));
}

// The next float up, past both zeros.
__device__ __forceinline__ float next_up(float v) {
  const int b = __float_as_int(v + 0.0f);
  return __int_as_float(b >= 0 ? b + 1 : b - 1);
}

// Loads that stay where they are written: ahead of the work that hides them.
__device__ __forceinline__ int load_now(const int *p) {
  int v;
  asm volatile("ld.global.s32 %0, [%1];" : "=r"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float load_now(const float *p) {
  float v;
  asm volatile("ld.global.f32 %0, [%1];" : "=f"(v) : "l"(p));
  return v;
}
__device__ __forceinline__ float load_now(const __nv_bfloat16 *p) {
  unsigned short v;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return __uint_as_float((unsigned)v << 16);
}
__device__ __forceinline__ float load_now(const __half *p) {
  unsigned short v;
  asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
  return __half2float(__ushort_as_half(v));
}

// Floats as integers of the same order, and back.
__device__ __forceinline__ int ordered(float v) {
  const int b = __float_as_int(v);
  return b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float unordered(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }

// A value that at least k <= 32 N of the warp's 32 N values reach and few
// more do.  Few: the greatest are taken off one after the other; else
// bisection, ended a little early.  Values are ordered integers.
constexpr int kNone = (int)0x80000000;  // below all of them
template <int N>
__device__ __forceinline__ int warp_kth(int *x, int k) {
  if (N == 1 && k <= 8) {
    int top, c = 0;
    do {
      top = __reduce_max_sync(0xffffffffu, x[0]);
      c += __popc(__ballot_sync(0xffffffffu, x[0] == top));
      if (x[0] == top) x[0] = kNone;
    } while (c < k);
    return top;
  }
  int lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) lo = min(lo, x[i]), hi = max(hi, x[i]);
  lo = __reduce_min_sync(0xffffffffu, lo);  // all values reach lo
  hi = __reduce_max_sync(0xffffffffu, hi);
  while (lo < hi) {
    const int mid = lo + (int)(((unsigned)hi - (unsigned)lo + 1u) >> 1);
    int c = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) c += x[i] >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= k) {
      lo = mid;
      if (c <= k + (k >> 3)) break;
    } else {
      hi = mid - 1;
    }
  }
  return lo;
}
// Such a value as a float: -inf when it lies below all logits.
__device__ __forceinline__ float as_bound(int v) { return unordered(max(v, (int)0x807fffff)); }

// The upper half of a sort key as an ordered integer; an empty key is kNone.
__device__ __forceinline__ int key_order(unsigned long long key) { return (int)(unsigned)(key >> 32) ^ kNone; }

// Sorts the warp's 32 keys, descending.
__device__ __forceinline__ unsigned long long warp_sort(unsigned long long key) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int size = 2; size <= 32; size *= 2)
#pragma unroll 1
    for (int s = size / 2; s > 0; s /= 2) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, s);
      const bool greater = ((lane & s) == 0) == ((lane & size) == 0);
      key = (other > key) == greater ? other : key;
    }
  return key;
}

// The place among n keys of one of them: the number of greater keys.
__device__ __forceinline__ int place_by_counting(const unsigned long long *cand, int n, unsigned long long key) {
  int at = n & 1 ? cand[n - 1] > key : 0;
#pragma unroll 4
  for (int j = 0; j + 1 < n; j += 2) {
    const ulonglong2 v = *reinterpret_cast<const ulonglong2 *>(cand + j);
    at += (v.x > key) + (v.y > key);
  }
  return at;
}
// The same among sorted runs of 32, by bisection in each.
__device__ __noinline__ int place_in_runs(const unsigned long long *cand, int n, unsigned long long key) {
  int at = 0;
#pragma unroll 2
  for (int r = 0; r < n; r += 32) {
    const unsigned long long *run = cand + r;
    int p = 0;
#pragma unroll
    for (int h = 16; h > 0; h /= 2)
      if (run[p + h - 1] > key) p += h;
    at += p + (run[p] > key);
  }
  return at;
}

// Writes the k greatest of n keys (k <= n; ids and log p, in order).  A key's
// place is found by counting the greater ones when the keys are few (n^2 / 2
// wide loads), else in sorted runs of 32 (n^2 / 5 loads, and the sorts).  The
// whole block calls it; room for a multiple of 32.
template <int NT>
__device__ __forceinline__ void put_greatest(unsigned long long *cand, int n, int k, int *ids, float *lps,
                                             const ScoreArgs &a, float m, float s, float ls) {
  const int t = threadIdx.x;
  const bool runs = n > 96;
  if (runs) {
    for (int i = t; i < (n + 31) / 32 * 32; i += NT) cand[i] = warp_sort(i < n ? cand[i] : 0);
    __syncthreads();
  }
  for (int i = t; i < n; i += NT) {
    const unsigned long long key = cand[i];
    const int at = runs ? place_in_runs(cand, n, key) : place_by_counting(cand, n, key);
    if (at < k && key) {
      ids[at] = key_id(key);
      lps[at] = log_p(a, key_logit(key), m, s, ls);
    }
  }
}

// Candidates held at most.  128 threads take rows with up to kFewTop
// alternatives, 256 those with more.
constexpr int kFewTop = 32;
constexpr int max_cap(int nt) { return nt == 128 ? 512 : 2048; }

// What the block's threads share of a row's candidates.
struct Pool {
  unsigned long long *key;  // cap of them
  int *n;                   // collected (may pass cap)
  int *ge;
  int *bound;  // one a warp
  int cap;
};

// Thins out a pool of n <= N NT candidates: those stay that reach the least of
// the values which each warp's share of k of its part of them reaches, at
// least k in all.  Returns that value.  The whole block calls it, after a
// barrier.
template <int NT, int N>
__device__ __noinline__ float thin_out(const Pool p, int n, int k) {
  constexpr int NW = NT / 32;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  unsigned long long own[N];
  int x[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int j = i * NT + lane * NW + wid;  // spread evenly over the warps
    own[i] = j < n ? p.key[j] : 0;
    x[i] = key_order(own[i]);
  }
  const int b = warp_kth<N>(x, (k + NW - 1) / NW);
  if (lane == 0) p.bound[wid] = b;
  __syncthreads();
  const int tau = __reduce_min_sync(0xffffffffu, p.bound[lane % NW]);
  if (threadIdx.x == 0) *p.n = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool keep = own[i] && key_order(own[i]) >= tau;
    const unsigned all = __ballot_sync(0xffffffffu, keep);
    if (!all) continue;
    int at = 0;
    if (lane == 0) at = atomicAdd(p.n, __popc(all));
    at = __shfl_sync(0xffffffffu, at, 0) + __popc(all & ((1u << lane) - 1));
    if (keep) p.key[at] = own[i];
  }
  __syncthreads();
  return as_bound(tau);
}

// A value that at least k of n keys reach and few more do, by one warp; -inf when n < k.
__device__ __noinline__ float about_kth(const unsigned long long *key, int n, int k) {
  if (n < k) return -INFINITY;
  const int lane = threadIdx.x & 31;
  int lo = 0x7fffffff, hi = kNone;
  for (int i = lane; i < n; i += 32) lo = min(lo, key_order(key[i])), hi = max(hi, key_order(key[i]));
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  while (lo < hi) {
    const int mid = lo + (int)(((unsigned)hi - (unsigned)lo + 1u) >> 1);
    int c = 0;
    for (int i = lane; i < n; i += 32) c += key_order(key[i]) >= mid;
    c = __reduce_add_sync(0xffffffffu, c);
    if (c >= k) {
      lo = mid;
      if (c <= k + (k >> 2) + 2) break;
    } else {
      hi = mid - 1;
    }
  }
  return as_bound(lo);
}

template <int NT>
__device__ __forceinline__ float thin_out(const Pool p, int n, int k) {
  if (n <= NT) return thin_out<NT, 1>(p, n, k);
  if (NT == 128 || n <= 4 * NT) return thin_out<NT, 4>(p, n, k);
  return thin_out<NT, max_cap(NT) / NT>(p, n, k);
}

// f(z, id) for this thread's logits >= least of `words` words a thread, the
// first of them w0 + thread; word(w) gives the staged or loaded word w.
template <typename E, int NT, class Get, class F>
__device__ __forceinline__ void each_logit(const Slice<E, NT> &s, int w0, int words, float least, Get word, F f) {
  for (int j = 0; j < words; ++j) {
    const int w = w0 + j * NT + (int)threadIdx.x;
    if (w >= s.n) break;
    const uint4 q = word(w);
    if (!(Word<E>::template max<1>(&q) >= least)) continue;
    const E *p = reinterpret_cast<const E *>(&q);
    for (int k = 0; k < Word<E>::kN; ++k) {
      const float z = Word<E>::one(p + k);
      const int id = s.id0(w) + k;
      if (z >= least && id >= 0 && id < s.V) f(z, id);
    }
  }
}

// More candidates than the pool holds (rows of few values, or ascending
// ones): the pool becomes between k and `few` keys that hold the k greatest
// of the slice's words [w0, w0 + words * NT), by bisection over whole keys
// from `tau` on; each reading takes the words again.  Returns the value they
// all reach.  The whole block calls it, after a barrier.
template <typename E, int NT, class Get>
__device__ __noinline__ float cut_out(const Pool p, const Slice<E, NT> s, int w0, int words, float tau, int k, int few,
                                      Get word) {
  const int t = threadIdx.x;
  unsigned long long lo = sort_key(tau, INT_MAX), hi = ~0ull;
  while (lo < hi) {  // a row with NaNs may have fewer than k numbers: it ends all the same
    const unsigned long long mid = lo + ((hi - lo - 1) >> 1) + 1;
    __syncthreads();
    if (t == 0) *p.ge = 0;
    __syncthreads();
    int g = 0;
    each_logit(s, w0, words, key_logit(mid), word, [&](float z, int id) { g += sort_key(z, id) >= mid; });
    g = __reduce_add_sync(0xffffffffu, g);
    if ((t & 31) == 0 && g) atomicAdd(p.ge, g);
    __syncthreads();
    g = *p.ge;
    if (g < k) {
      hi = mid - 1;
    } else {
      lo = mid;
      if (g <= few) break;
    }
  }
  if (t == 0) *p.n = 0;
  __syncthreads();
  each_logit(s, w0, words, key_logit(lo), word, [&](float z, int id) {
    if (sort_key(z, id) >= lo) p.key[atomicAdd(p.n, 1)] = sort_key(z, id);
  });
  __syncthreads();
  return key_logit(lo);
}

// Rows stream through a ring of D chunks of shared memory: a thread waits for
// its own words, takes them up, and sends for the chunk D further on, of this
// row or the next.
//
// Alternatives are found on the way, in one reading.  From the first chunk's
// maxima comes a value tau that at least k logits reach; what reaches it is a
// candidate.  In later chunks only logits above tau can be alternatives, since
// equal ones have greater ids than k others.  Each time the row has grown
// `grow` times the block meets and, when the candidates are half again as
// many as k, raises tau to about their k-th greatest and drops the rest; in
// between its warps run on their own.  More candidates than the
// buffer holds are cut out exactly: those of the first chunk from its staged
// words (rows of few values, or masked but for fewer than k), those of a row
// whose logits keep rising by reading it again.  What remains is ordered at
// the row's end.
//
// A row over a cluster (few rows) has each slice find its own candidates;
// those that reach the least of the slices' about ceil(k / C)-th greatest are
// at least k, and go to rank 0, which orders them.
template <typename E, int NT, int D, bool TOPK, bool ENT>
__global__ void __launch_bounds__(NT, (NT == 128 ? 8 : 4) - TOPK) snai_score(const ScoreArgs a) {
  constexpr int NW = NT / 32, kWide = kChunk * NT, kN = Word<E>::kN;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Stat part[2][NW];
  __shared__ Slip slip[2];
  __shared__ int bound[2][NW], n_cand[2], n_ge;
  __shared__ int n_lead[2];  // by row: the others read a row's count while rank 0 is already at the next one
  uint4 *ring = reinterpret_cast<uint4 *>(smem);
  // candidates, then (rank 0 of a cluster) those of all slices
  unsigned long long *cand = reinterpret_cast<unsigned long long *>(smem + D * kWide * 16);
  unsigned long long *gath = cand + a.cap;
  int par = 0;
  auto pool = [&] { return Pool{cand, &n_cand[par], &n_ge, bound[par], a.cap}; };
  const int t = threadIdx.x, lane = t & 31, wid = t >> 5;
  const int C = a.in.C;
  const unsigned rank = C > 1 ? cluster_ctarank() : 0;
  const int step = gridDim.x / C;
  const int chunks = (a.in.wps + kWide - 1) / kWide;
  const float above = kAbove / a.c;

  Slice<E, NT> cur, ahead;  // the row in work, the row being sent for
  int r = blockIdx.x / C, ra = r, ca = 0, slot = 0;
  cur.set(a.in, r, rank);
  ahead = cur;
  auto send = [&](uint4 *to) {  // the next chunk of the stream, a group of its own
    if (ra < a.in.rows) {
      ahead.load_chunk(ca, to);
      if (++ca == chunks) {
        ca = 0;
        if (ra + step < a.in.rows) ahead.next(a.in, ra, step, rank);
        ra += step;
      }
    }
    ahead.commit();
  };
  int tok[kMaxList / NT];
  auto next_tokens = [&](int row) {
#pragma unroll
    for (int i = 0; i < kMaxList / NT; ++i) {
      const int j = i * NT + t;
      tok[i] = j < a.n_tok ? load_now(a.tokens + (long long)row * a.n_tok + j) : -1;
    }
  };
  if (rank == 0 && wid * 32 < a.n_tok) next_tokens(r);
  for (int i = 0; i < D; ++i) send(ring + i * kWide);
  for (; r < a.in.rows; par ^= 1) {
    // the tokens' logits, read beside the row's copies; the next row's tokens
    float zt[kMaxList / NT];
    bool in[kMaxList / NT];
    if (rank == 0 && wid * 32 < a.n_tok) {
#pragma unroll
      for (int i = 0; i < kMaxList / NT; ++i) {
        in[i] = tok[i] >= 0 && tok[i] < a.in.V;
        zt[i] = in[i] ? load_now(cur.at(tok[i])) : 0.f;
      }
      if (r + step < a.in.rows) next_tokens(r + step);
    }
    Running<E, ENT, false> run;
    float tau = -INFINITY, least = -INFINITY;  // of a chunk's logits, those from `least` on are candidates
    int meet = a.grow - 1;                     // the chunk after which the block meets next
    for (int c = 0; c < chunks; ++c) {
      uint4 *at = ring + slot * kWide;
      slot = slot + 1 == D ? 0 : slot + 1;
      copies_wait<D - 1>();
      uint4 q[kChunk];
      cur.chunk(c, at, q);
      float wm[kChunk];
#pragma unroll
      for (int j = 0; j < kChunk; ++j) wm[j] = Word<E>::template max<1>(q + j);
      const float cm = max_nan(max_nan(wm[0], wm[1]), max_nan(wm[2], wm[3]));
      run.add(q, cm, a.c, above);
      if (TOPK) {
        if (c == 0) {
          // Each warp gives a value that its share of the k groups reach, of
          // groups of four words, two, or one; all reach the least of these.
          constexpr int kFew = 8;
          const int k = (a.top_k + NW - 1) / NW;
          int b;
          if (k <= kFew) {
            int v = ordered(cm);
            b = warp_kth<1>(&v, k);
          } else if (k <= 2 * kFew) {
            int v[2] = {ordered(max_nan(wm[0], wm[1])), ordered(max_nan(wm[2], wm[3]))};
            b = warp_kth<2>(v, k);
          } else {
            int v[4] = {ordered(wm[0]), ordered(wm[1]), ordered(wm[2]), ordered(wm[3])};
            b = warp_kth<4>(v, k);
          }
          if (lane == 0) bound[par][wid] = b;
          if (t == 0) n_cand[par] = 0;
          __syncthreads();
          tau = least = as_bound(__reduce_min_sync(0xffffffffu, bound[par][lane % NW]));
        }
        if (cm >= least) {
          // this thread's hits as bits, room for them, then their keys
          unsigned hits = 0;
          const unsigned lim = Word<E>::limit(least);
#pragma unroll
          for (int j = 0; j < kChunk; ++j)
            if (wm[j] >= least && c * kWide + j * NT + t < cur.n) hits |= Word<E>::reach(q[j], lim) << (j * kN);
          for (int p = hits ? atomicAdd(&n_cand[par], __popc(hits)) : 0; hits; hits &= hits - 1, ++p) {
            const int b = __ffs(hits) - 1, j = b / kN, k = b % kN, id = cur.id0(c * kWide + j * NT + t) + k;
            const float z = Word<E>::one(reinterpret_cast<const E *>(at + j * NT + t) + k);
            // the masked filling behind the row's ends is no logit: an empty key
            if (p < a.cap) cand[p] = id >= 0 && id < cur.V ? sort_key(z, id) : 0;
          }
        }
        if (c + 1 < chunks && (c == meet || (c == 0 && tau == -INFINITY))) {
          __syncthreads();
          const int n = n_cand[par];
          __syncthreads();
          if (n > a.cap)
            tau = c == 0 ? cut_out<E, NT>(pool(), cur, 0, kChunk, tau, a.top_k, a.soft, [at](int w) { return at[w]; })
                         : cut_out<E, NT>(pool(), cur, 0, (c + 1) * kChunk, tau, a.top_k, a.soft,
                                          [cur](int w) { return cur.fetch(w); });
          else if (n > a.soft)
            tau = fmaxf(tau, thin_out<NT>(pool(), n, a.top_k));
          if (c == meet) meet = a.grow * (meet + 1) - 1;
        }
        least = next_up(tau);
      }
      if (c + 1 < chunks) send(at);
    }
    Stat st = combine_lanes<ENT, false>(run.get(), 32, a.c);
    if (lane == 0) part[par][wid] = st;
    __syncthreads();
    uint4 *last = ring + (slot == 0 ? D - 1 : slot - 1) * kWide;  // the row's last chunk, not yet sent for again
    int n = TOPK ? n_cand[par] : 0;
    if (TOPK && n > a.cap) {
      if (chunks == 1)
        cut_out<E, NT>(pool(), cur, 0, kChunk, tau, a.top_k, a.soft, [last](int w) { return last[w]; });
      else
        cut_out<E, NT>(pool(), cur, 0, chunks * kChunk, tau, a.top_k, a.soft, [cur](int w) { return cur.fetch(w); });
      n = n_cand[par];
    } else if (TOPK && n > 128 && n > 3 * a.top_k) {  // cheaper than ordering them all
      thin_out<NT>(pool(), n, a.top_k);
      n = n_cand[par];
    }
    send(last);
    if (C > 1) {
      if (wid == 0) {
        st = combine_lanes<ENT, false>(part[par][lane % NW], NW, a.c);
        if (TOPK)
          tau = st.s != st.s ? INFINITY
                             : about_kth(cand, n, (a.top_k + C - 1) / C);
        if (lane == 0) slip[par].st = st, slip[par].tau = tau, n_lead[par] = 0;
      }
      cluster_sync_all();
      const bool on = lane % 16 < C;
      st = combine_lanes<ENT, false>(on ? peer_stat(&slip[par], lane % 16) : no_stat(), 16, a.c);
      if (TOPK) {
        tau = on ? __uint_as_float(ld_cluster_u32(mapa_shared(smem_u32(&slip[par].tau), lane % 16))) : INFINITY;
        tau = -warp_max_nan(-tau);
      }
    } else if (TOPK || wid * 32 < max(a.n_tok, 1)) {
      st = combine_lanes<ENT, false>(part[par][lane % NW], NW, a.c);
    }
    // c is off by up to half a step, which is T off by as much and moves
    // log S by that times the mean of d: known where W is
    const float log_s = logf(st.s), ls = ENT ? fmaf(a.off, __fdividef(st.w, st.s), log_s) : log_s;
    if (rank == 0 && t < max(a.n_tok, 1)) {
#pragma unroll
      for (int i = 0; i < kMaxList / NT; ++i) {
        const int j = i * NT + t;
        if (j < a.n_tok)
          a.logprob[(long long)r * a.n_tok + j] = in[i] ? log_p(a, zt[i], st.m, st.s, ls) : 0.f;
      }
      if (ENT && t == 0 && a.entropy) a.entropy[r] = st.s == 0.f ? 0.f : log_s - kLn2 * st.w / st.s;
    }
    if (TOPK) {
      int *ids = a.top_ids + (long long)r * a.top_k;
      float *lps = a.top_logprob + (long long)r * a.top_k;
      if (st.s != st.s) {
        if (rank == 0)
          for (int i = t; i < a.top_k; i += NT) ids[i] = -1, lps[i] = NAN;
      } else if (C == 1) {
        put_greatest<NT>(cand, n, a.top_k, ids, lps, a, st.m, st.s, ls);
      } else {
        const uint32_t to_n = mapa_shared(smem_u32(&n_lead[par]), 0), to = mapa_shared(smem_u32(gath), 0);
        const uint32_t to_ge = mapa_shared(smem_u32(&n_ge), 0);
        unsigned long long lo = sort_key(tau, INT_MAX), hi = ~0ull;
        auto gather = [&] {
          for (int i = t; i < n; i += NT)
            if (cand[i] >= lo) {
              const unsigned p = atom_cluster_add_u32(to_n, 1);
              if (p < (unsigned)a.cap) st_cluster_u64(to + 8 * p, cand[i]);
            }
        };
        gather();
        cluster_sync_all();
        int m = (int)ld_cluster_u32(to_n);
        if (m > a.cap) {  // ties over several slices: bisect
          while (lo < hi) {
            const unsigned long long mid = lo + ((hi - lo - 1) >> 1) + 1;
            cluster_sync_all();
            if (t == 0) n_ge = 0, n_lead[par] = 0;
            cluster_sync_all();
            int g = 0;
            for (int i = t; i < n; i += NT) g += cand[i] >= mid;
            g = __reduce_add_sync(0xffffffffu, g);
            if (lane == 0 && g) atom_cluster_add_u32(to_ge, (unsigned)g);
            cluster_sync_all();
            m = (int)ld_cluster_u32(to_ge);
            if (m < a.top_k) {
              hi = mid - 1;
            } else {
              lo = mid;
              if (m <= a.cap) break;
            }
          }
          gather();
          cluster_sync_all();
        }
        if (rank == 0) put_greatest<NT>(gath, m, a.top_k, ids, lps, a, st.m, st.s, ls);
      }
    }
    if (r + step < a.in.rows) cur.next(a.in, r, step, rank);
    r += step;
  }
  if (C > 1) cluster_sync_all();  // others may still read this CTA's slip
}

// ---- row gradients ----

struct RowGradArgs {
  Rows in;
  const int *ids;     // [rows][n] tokens, or teacher ids
  const float *vals;  // [rows][n] their gradients, or teacher values
  int n;
  float c;           // log2(e) / T
  float inv_t_f;
  double inv_t;      // 1 / T
  // the 1 / T that c, rounded, stands for, and the 1 that a label's exponents
  // do: with them a loss is that of a temperature off by half a step of fp32,
  // and not the difference of two
  double inv_t_z, one_z;
  const float *g_entropy;
  const int *labels;
  const float *row_grad;
  double t, a;  // temperature, label weight
  int rest;
  float *loss;
  void *grad;
  long long grad_ld;
};

__device__ __forceinline__ void copy4(void *dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ double warp_sum_d(double v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// exp(x) in 64 bits for x <= 0 to 1e-11: 2^n times 1 + f + f^2 / 2 + f^3 P(f),
// P of the fifth degree through (exp(f) - 1 - f - f^2 / 2) / f^3 at the six
// Chebyshev nodes of [-ln2 / 2, ln2 / 2] (0 below -700; a NaN stays one, and
// what is not <= 0 by rounding or mistake is exact enough up to 700).  The
// Taylor series of as many terms is off by 2e-10, which shows where a list
// leaves 1e-8 of 1; one of three terms more cost 3 to 6 % of a call.
__device__ __forceinline__ double exp_d(double x) {
  if (!(x > -700.0)) return x != x ? x : 0.0;
  if (x > 700.0) return INFINITY;
  const double n = rint(x * 1.4426950408889634074);
  const double f = fma(-n, 0.69314718055994530942, x);
  const double f2 = f * f;
  const double lo = fma(f, fma(f, 0.16666666681659179, 0.5), 1.0);
  const double hi =
      fma(f, fma(f, fma(f, fma(f, 2.4851337915360752e-05, 0.00019891030654370327), 0.0013888866451042758),
                 0.008333310889582076),
          0.041666666681655085);
  const double e = fma(f, fma(f2 * f, hi, lo), 1.0);
  return e * __hiloint2double((1023 + (int)n) << 20, 0);
}

// Barrier of the cluster behind one thread's writes (the caller's thread 0,
// which has fenced them): the other threads' gradient stores need not have
// drained, as a release by every thread would have them.
__device__ __forceinline__ void fence_cluster() { asm volatile("fence.acq_rel.cluster;" ::: "memory"); }
__device__ __forceinline__ void cluster_meet() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// MODE 0: the gradient of scores.  With x_i = d_i / ln 2, G the sum of the
// row's token gradients and g_H the entropy's (EXTRA: when there is one):
//   grad_i = e_i (alpha + beta x_i) + (sum of g_j of the tokens equal to i) / T,
//   alpha = (g_H ln2 W / S - G) / (S T),  beta = -g_H ln2 / (S T).
// MODE 1: distillation, q_j the teacher's weights:
//   grad_i = e_i alpha + gamma softmax(z)_i - what the list and the label take.
// EXTRA: labels at T != 1, whose softmax needs exponentials of its own (1), or
// at T = 2 or 4 the squares (2) or fourth powers (3) of those at hand
// (8192 x 16384, 64 entries: 191 us against 215 with exponentials of their
// own; 4096 x 32000 bf16: 135 against 177).  With `rest` the listed logits
// are taken out of the staged row (each by the thread that owns its word,
// which finds it in a list of its own), so that the unlisted mass is a sum of
// its own: 1 - the listed would lose a confident student's.
//
// The first NT threads stage the row and take it through both passes; 32 or
// 64 more, the entry threads, have the list: they work beside pass A, with the
// entries' logits read from global memory, so that what a row costs the others
// is one barrier (`rest`: two) and the scalars, which every warp then works
// out.  Pass B writes the terms that every element has; the entries' ids get
// theirs from the entry threads one row later, behind the next row's barrier,
// when all owners have written the base.  (Entries held by threads that also
// take the row took 46 us where these first took 34 (now 31), at 1024 x 16384 with 64 entries
// and labels: their chain of dependent steps is as long as both passes.)  An
// id listed more than once is handled by its first entry, in the order of the
// list: no atomics.  The entries' weights and the loss are held in 64 bits: a
// handful of values a row, and a loss that is a small difference of large
// terms.
constexpr float kNoRest = 1074.8f;  // 745 / ln 2: e^-745 is the least number of 64 bits
constexpr int kMaxEntryWarps = 2;  // more would cost the third CTA of an SM its registers
template <typename E, int NT, int MODE, int EXTRA>
__global__ void __launch_bounds__(NT + 32 * kMaxEntryWarps, NT == 128 ? 5 : 3) snai_row_grad(const RowGradArgs a) {
  constexpr int NW = NT / 32, kN = Word<E>::kN, kWide = kChunk * NT;
  constexpr bool ENT = MODE == 0 && EXTRA, LABEL1 = MODE == 1 && EXTRA;
  constexpr int SQ = LABEL1 ? EXTRA - 1 : 0;  // squarings that make exp(d) of exp(d / T)
  // aligned: else a warp's 512 bytes take five rows of banks (2048 x 131072
  // with the rest 376 us, and 435 on 16 bytes)
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ Stat part[2][NW], listed[2][kMaxEntryWarps];
  // by entry warp: the sums of q (MODE 0: g) and of q (log q - (z - top) / T), and top
  __shared__ double sum_q[2][kMaxEntryWarps], sum_kl[kMaxEntryWarps];
  __shared__ float list_top[kMaxEntryWarps];
  __shared__ float label_z, scal[2];  // the label's logit; g_entropy or row_grad of two rows
  __shared__ Slip slip[2];
  uint4 *buf = reinterpret_cast<uint4 *>(smem);
  const bool rest = MODE == 1 && a.rest;
  const int n = a.n, ne = n + (MODE == 1 && a.labels ? 1 : 0), cap = (ne + 3) & ~3;
  // lists: ids and values of two rows; the entries' weights and logits; the
  // pending gradients; (rest) the owners' links, and their heads
  int *ids2 = reinterpret_cast<int *>(smem + (size_t)a.in.wps * 16);
  float *vals2 = reinterpret_cast<float *>(ids2 + 2 * cap);
  float *wt = vals2 + 2 * cap, *zl = wt + cap, *fix = zl + cap;
  int *fix_id = reinterpret_cast<int *>(fix + cap);
  int2 *link = reinterpret_cast<int2 *>(fix_id + cap);
  int *head = reinterpret_cast<int *>(link + cap);
  const int t = threadIdx.x, lane = t & 31, wid = t >> 5;
  const bool entry = wid >= NW;
  const int et = t - NT, ew = wid - NW, nwe = ((int)blockDim.x - NT) / 32, nte = nwe * 32;
  const int C = a.in.C;
  const unsigned rank = C > 1 ? cluster_ctarank() : 0;
  const int step = gridDim.x / C;
  const int V = a.in.V;
  auto valid = [&](int id) { return id >= 0 && id < V; };
  auto load_lists = [&](int row, int b) {
    for (int j = et; j < n; j += nte) {
      copy4(ids2 + b * cap + j, a.ids + (long long)row * n + j);
      copy4(vals2 + b * cap + j, a.vals + (long long)row * n + j);
    }
    if (ne > n && et == n % nte) copy4(ids2 + b * cap + n, a.labels + row);
    if (et == 0) {
      if (ENT) copy4(&scal[b], a.g_entropy + row);
      if (MODE == 1 && a.row_grad) copy4(&scal[b], a.row_grad + row);
    }
  };
  Slice<E, NT> cur;
  int r = blockIdx.x / C;
  cur.set(a.in, r, rank);
  const int chunks = (a.in.wps + kWide - 1) / kWide, cps = (chunks + kStages - 1) / kStages;
  if (entry) {
    for (int j = et; j < cap; j += nte) ids2[cap + j] = fix_id[j] = -1;
    for (int j = ne + et; j < cap; j += nte) ids2[j] = -1;
    load_lists(r, 0);
    cur.commit();
    copies_wait<0>();
  } else {
    for (int s = 0; s < kStages; ++s) cur.load(s, cps, buf);
    head[t] = -1;
  }
  __syncthreads();
  int par = 0;

  // The scalars of a row, by every warp behind the row's barrier.  S and S1 are
  // relative to m.  With `rest` the unlisted sum su is relative to the unlisted
  // maximum mu, and stays so: relative to a listed one 87 T above it would be 0.
  // Pass B, which then gives the unlisted ids' gradients alone, takes its
  // exponentials relative to mu too (else mu is m).
  float m, mu, S, S1, su, inv_s, inv_s1, alpha, beta, gamma, kt, ky, mass, rest_k;
  double rr, q_all;
  auto scalars = [&](float sc, int y) {
    Stat st = combine_lanes<ENT, LABEL1>(part[par][lane % NW], NW, a.c);
    if (C > 1) {
      if (t == 0) {
        slip[par].st = st;
        fence_cluster();
      }
      __syncwarp();
      cluster_meet();
      st = combine_lanes<ENT, LABEL1>(lane % 16 < C ? peer_stat(&slip[par], lane % 16) : no_stat(), 16, a.c);
    }
    q_all = sum_q[par][0];
    if (nwe > 1) q_all += sum_q[par][1];
    mu = st.m, su = st.s;
    float f = 1.f;  // 2^((mu - m) c)
    if (rest) {
      Stat lst = lane % 2 < nwe ? listed[par][lane % 2] : no_stat();
      const float both = max_nan(mu, warp_max_nan(lst.m));
      f = ex2(cut((mu - both) * a.c));
      if (LABEL1) st.s1 *= ex2(cut((mu - both) * kLog2E));
      rebase<false, LABEL1>(lst, both, a.c);
      lst = combine_lanes<false, LABEL1>(lst, 2, a.c);
      st.m = both;
      st.s = fmaf(su, f, lst.s);
      if (LABEL1) st.s1 += lst.s1;
    }
    m = st.m;
    S = st.s;
    S1 = LABEL1 ? st.s1 : S;
    inv_s = S == 0.f ? 0.f : 1.f / S;
    inv_s1 = LABEL1 ? (S1 == 0.f ? 0.f : 1.f / S1) : inv_s;
    beta = gamma = kt = ky = mass = rest_k = 0.f;
    rr = 0;
    if (MODE == 0) {
      const float gh = ENT ? sc : 0.f, k = inv_s * a.inv_t_f;
      alpha = -(float)q_all * k;
      if (ENT) alpha += gh * kLn2 * st.w * inv_s * k, beta = -gh * kLn2 * k;
    } else {
      // Has the student any unlisted probability in 64 bits?  su is 0 or at least 1.
      // All threads come to the same answer: rounded step by step, never contracted.
      bool some = su > 0.f;
      if (rest && f == 0.f)
        some = some && __fadd_rn(__fmul_rn(m - mu, a.c), __fsub_rn(__log2f(S), __log2f(su))) < kNoRest;
      rr = rest && some ? fmax(0.0, 1.0 - q_all) : 0.0;
      mass = (float)(q_all + rr);
      rest_k = rr > 0.0 ? (float)rr / su : 0.f;  // times an unlisted e_i: what the teacher's rest gives to i
      kt = sc * (float)((1.0 - a.a) * a.t);
      ky = y >= 0 ? sc * (float)a.a : 0.f;
      f *= inv_s;  // times e_i: p_i
      alpha = kt * (mass * f - rest_k);
      if (LABEL1)
        gamma = ky * (rest ? ex2(cut((mu - m) * kLog2E)) * inv_s1 : inv_s1);
      else
        alpha += ky * f;
    }
  };

  if (entry) {
    E *before = nullptr;  // the row whose entries' gradients are pending
    auto entry_sync = [&] {
      if (nwe > 1)
        asm volatile("bar.sync 1, %0;" ::"r"(nte) : "memory");
      else
        __syncwarp();
    };
    // the thread that owns an id's word, when it is in this slice; equal for equal ids
    auto hash = [&](int id) { return (unsigned)(id - cur.base + (1 << 20)) / kN % NT; };
    auto store_pending = [&] {
      if (before)
        for (int j = et; j < ne; j += nte)
          if (fix_id[j] >= 0) Word<E>::put(before + fix_id[j], fix[j]);
    };
    for (; r < a.in.rows; r += step, par ^= 1) {
      const int *ids = ids2 + par * cap;
      const float *vals = vals2 + par * cap;
      if (r + step < a.in.rows) load_lists(r + step, par ^ 1);
      cur.commit();
      const int y = ne > n && valid(ids[n]) ? ids[n] : -1;
      const float sc = ENT || (MODE == 1 && a.row_grad) ? scal[par] : 1.f;
      bool any = ENT && et == 0 && sc != 0.f;  // anything but padding in the row?
      unsigned firsts = 0, again = 0;          // by entry of this thread: the id's first; listed again later
      // the entries' logits are asked for first (one a thread without waiting)
      const float z0 = et < ne && valid(ids[et]) ? load_now(cur.at(ids[et])) : -INFINITY;
      for (int j = et; j < ne; j += nte) {
        const int id = ids[j];
        if (!valid(id)) continue;
        any = true;
        link[j] = make_int2(cur.local(id), atomicExch(&head[hash(id)], j));
      }
      // behind the barrier owners find the listed logits among their words,
      // and entries those that name the same id
      if (rest)
        __syncthreads();
      else
        entry_sync();
      for (int j = et, i = 0; j < ne; j += nte, ++i) {
        const int id = ids[j];
        if (!valid(id)) continue;
        firsts |= 1u << i;
        for (int l = head[hash(id)]; l >= 0; l = link[l].y)
          if (ids[l] == id && l != j) {
            if (l < j) firsts &= ~(1u << i);
            if (l > j && l < n) again |= 1u << i;
          }
      }
      double lse = 0;
      if (MODE == 1 && !rest) {  // the teacher's log normaliser, by every entry warp
        float tm = -INFINITY, s = 0.f;
        for (int j = lane; j < n; j += 32)
          if (valid(ids[j])) tm = max_nan(tm, vals[j]);
        tm = warp_max_nan(tm);
        for (int j = lane; j < n; j += 32)
          if (valid(ids[j]) && vals[j] != -INFINITY) s += expf((float)(((double)vals[j] - tm) * a.inv_t));
        s = warp_sum(s);
        // log s = ls + log(s exp(-ls)), the second to its first order: an error here is one of the whole loss
        const float ls = logf(s);
        lse = tm == -INFINITY ? 0.0 : tm * a.inv_t + ls + ((double)s * exp_d(-(double)ls) - 1.0);
      }
      for (int j = et; j < ne; j += nte) zl[j] = j == et ? z0 : valid(ids[j]) ? Word<E>::one(cur.at(ids[j])) : -INFINITY;
      // logits are taken relative to the warp's greatest, so that a row of the type's lowest values keeps its differences
      float top = 0.f;
      if (MODE == 1) {
        top = -INFINITY;
        for (int j = et; j < n; j += nte) top = max_nan(top, zl[j]);
        top = warp_max_nan(top);
        if (top == -INFINITY) top = 0.f;
      }
      double q_own = 0, kl_own = 0;
      Stat own = no_stat();
      for (int j = et, i = 0; j < n; j += nte, ++i) {
        const int id = ids[j];
        const float z = zl[j];
        double q = 0;
        if (MODE == 0) {
          if (valid(id)) q = vals[j];
        } else if (valid(id) && vals[j] != -INFINITY) {
          const double lq = rest ? (double)vals[j] : vals[j] * a.inv_t - lse;
          q = exp_d(lq);  // not fp32's: an entry of 1e-60 against a masked logit is an infinite loss all the same
          if (q != 0.0) kl_own += q * (lq - ((double)z - top) * a.inv_t_z);
        }
        q_own += q;
        wt[j] = (float)q;
        if (rest && (firsts >> i & 1)) {
          const float nm = max_nan(own.m, z);
          rebase<false, LABEL1>(own, nm, a.c);
          own.s += ex2(cut((z - nm) * a.c));
          if (LABEL1) own.s1 += ex2(cut((z - nm) * kLog2E));
        }
      }
      if (ne > n && et == n % nte) {
        wt[n] = 0.f;
        label_z = zl[n];
      }
      q_own = MODE == 0 ? (double)warp_sum((float)q_own) : warp_sum_d(q_own);
      if (MODE == 1) kl_own = warp_sum_d(kl_own);
      if (rest) own = combine_lanes<false, LABEL1>(own, 32, a.c);
      if (lane == 0) {
        sum_q[par][ew] = q_own;
        if (MODE == 1) sum_kl[ew] = kl_own, list_top[ew] = top;
        if (rest) listed[par][ew] = own;
      }
      copies_wait<0>();  // the next row's lists
      any = __syncthreads_or(any);
      store_pending();  // over the base that the row before's owners have written
      scalars(sc, y);
      if (a.grad) {
        for (int j = et, i = 0; j < ne; j += nte, ++i) {
          const int id = ids[j];
          fix_id[j] = any && (firsts >> i & 1) && cur.local(id) >= 0 ? id : -1;
          float q = wt[j];
          if (again >> i & 1)
            for (int l = j + 1; l < n; ++l)
              if (ids[l] == id) q += wt[l];
          const float z = zl[j], d = z - m;
          float g;
          if (MODE == 0) {
            const float x = cut(d * a.c);
            g = ex2(x) * fmaf(x, beta, alpha) + q * a.inv_t_f;
          } else {
            const float p = ex2(cut(d * a.c)) * inv_s;
            g = kt * (mass * p - (j < n ? q : rest_k * ex2(cut((z - mu) * a.c))));
            if (y >= 0) {
              const float p1 = LABEL1 ? ex2(cut(d * kLog2E)) * inv_s1 : p;
              g += ky * (id == y ? p1 - 1.f : p1);
            }
          }
          fix[j] = S != S ? NAN : z == -INFINITY ? 0.f : g;
        }
        before = static_cast<E *>(a.grad) + (long long)r * a.grad_ld;
      }
      if (MODE == 1 && et >= nte - 32 && rank == 0) {  // the loss, by the last entry warp
        // With `rest` S is taken again in 64 bits from its two parts, relative to
        // the greater one's maximum: no gap between them is lost, and log S and
        // the log of the unlisted sum come from the same terms.
        double all = S, gap = 0.0;  // what the listed maximum is above the unlisted one
        float ref = m, tops = 1.f;  // what `all` is relative to, and how much of it is exact: a term of each part
        if (rest && su > 0.f) {
          const Stat lst = combine_lanes<false, false>(lane % 2 < nwe ? listed[par][lane % 2] : no_stat(), 2, a.c);
          gap = ((double)lst.m - mu) * a.inv_t_z;
          const double x = exp_d(-fabs(gap));
          const bool above = lst.m > mu;
          all = above ? lst.s + x * su : su + x * lst.s;
          ref = above ? lst.m : mu;
          tops = lst.s > 0.f ? 1.f + (float)x : 1.f;
        }
        // every logarithm at once, a lane each; lane 0 has its own at hand and the loss is its
        const double logs = log(lane == 0 ? all : lane == 1 ? (double)su : lane == 2 ? (double)S1 : rr);
        auto log_of = [&](int i) { return __shfl_sync(0xffffffffu, logs, i); };
        double l = 0;
        if (S == 0.f) {
          l = q_all > 0 ? INFINITY : 0.0;
        } else {
          const double log_s = logs + kEx2Low * (1.f - __fdividef(tops, (float)all));
          if (rr > 0.0)  // the student's rest is the unlisted sum over all
            l = rr * (log_of(3) + (log_s - (log_of(1) + kEx2Low * (1.f - __fdividef(1.f, su)))) + fmax(gap, 0.0));
          for (int w = 0; w < nwe; ++w) l += sum_kl[w] + sum_q[par][w] * (((double)ref - list_top[w]) * a.inv_t_z);
          l += q_all * log_s;
        }
        l = a.a < 1.0 ? l * ((1.0 - a.a) * a.t * a.t) : 0.0;
        if (y >= 0) l += a.a * (label_z == -INFINITY ? INFINITY : ((double)m - label_z) * a.one_z + log_of(2));
        if (lane == 0) a.loss[r] = !any ? 0.f : S != S ? NAN : (float)l;
      }
      for (int j = et; j < ne; j += nte)
        if (valid(ids[j])) head[hash(ids[j])] = -1;
      entry_sync();  // what the entry warps share of a row is overwritten by the next
      if (r + step < a.in.rows) cur.next(a.in, r, step, rank);
    }
    __syncthreads();
    store_pending();
  } else {
    const float above = kAbove / fmaxf(a.c, LABEL1 ? kLog2E : 0.f);
    for (; r < a.in.rows; r += step, par ^= 1) {
      const bool more = r + step < a.in.rows;
      Slice<E, NT> nxt = cur;
      if (more) nxt.next(a.in, r, step, rank);
      const int label = ne > n ? ids2[par * cap + n] : -1, y = valid(label) ? label : -1;
      const float sc = ENT || (MODE == 1 && a.row_grad) ? scal[par] : 1.f;
      // the listed logits among this thread's words: two at hand, the others linked
      int e0 = -1, e1 = -1, others = -1;
      if (rest) {
        __syncthreads();
        others = head[t];
        if (others >= 0) {
          int2 l = others < n ? link[others] : make_int2(-1, link[others].y);
          e0 = l.x, others = l.y;
          if (others >= 0) l = link[others], e1 = others < n ? l.x : -1, others = l.y;
        }
      }
      const int c0 = e0 < 0 ? -1 : e0 / (kN * kWide), c1 = e1 < 0 ? -1 : e1 / (kN * kWide);
      // pass A
      Running<E, ENT, LABEL1, SQ> run;
#pragma unroll 1
      for (int s = 0; s < kStages; ++s) {
        if (!a.grad && more)  // no pass B: one group of the next row follows each stage
          copies_wait<kStages - 1>();
        else
          copies_wait(kStages - 1 - s);
#pragma unroll 1
        for (int c = s * cps; c < (s + 1) * cps && c < chunks; ++c) {
          if (rest) {
            if (c0 == c) Word<E>::put(reinterpret_cast<E *>(buf) + e0, -INFINITY);
            if (c1 == c) Word<E>::put(reinterpret_cast<E *>(buf) + e1, -INFINITY);
            for (int j = others; j >= 0;) {
              const int2 l = link[j];
              if (j < n && l.x >= 0 && l.x / (kN * kWide) == c) Word<E>::put(reinterpret_cast<E *>(buf) + l.x, -INFINITY);
              j = l.y;
            }
          }
          uint4 q[kChunk];
          cur.chunk(c, buf + c * kWide, q);
          run.add(q, Word<E>::template max<kChunk>(q), a.c, above);
        }
        if (!a.grad && more) nxt.load(s, cps, buf);
      }
      const Stat st = combine_lanes<ENT, LABEL1>(run.get(), 32, a.c);
      if (lane == 0) part[par][wid] = st;
      const bool any = __syncthreads_or(false);
      if (a.grad || C > 1) scalars(sc, y);
      if (a.grad) {
        // pass B
        E *out = static_cast<E *>(a.grad) + (long long)r * a.grad_ld;
        const bool vec = ((reinterpret_cast<uintptr_t>(out) + (long long)cur.base * (int)sizeof(E)) & 15) == 0;
        const f2 nm2 = pack2(-mu, -mu), c2 = pack2(a.c, a.c), l2 = pack2(kLog2E, kLog2E);
        const f2 al2 = pack2(alpha, alpha), be2 = pack2(beta, beta), ga2 = pack2(gamma, gamma);
#pragma unroll 1
        for (int s = 0; s < kStages; ++s) {
#pragma unroll 1
          for (int c = s * cps; c < (s + 1) * cps && c < chunks; ++c) {
            uint4 q[kChunk];
            cur.chunk(c, buf + c * kWide, q);
#pragma unroll
            for (int j = 0; j < kChunk; ++j) {
              f2 v[kN / 2];
              Word<E>::unpack(q[j], v);
#pragma unroll
              for (int k = 0; k < kN / 2; ++k) {
                const f2 d = add2(v[k], nm2);
                f2 x = mul2(d, c2);
                float u, w;
                unpack2(x, u, w);
                if (ENT) {
                  u = cut(u), w = cut(w);
                  x = pack2(u, w);
                }
                const f2 e = pack2(ex2(u), ex2(w));
                v[k] = mul2(e, ENT ? fma2(x, be2, al2) : al2);
                if (LABEL1) v[k] = fma2(at_one<SQ>(e, d, l2), ga2, v[k]);
              }
              q[j] = any ? Word<E>::pack(v) : make_uint4(0u, 0u, 0u, 0u);
            }
            const int w0 = c * kWide + t;
            E *o = out + cur.id0(w0);
            if (vec && c * kWide >= cur.lo && (c + 1) * kWide <= cur.hi) {
#pragma unroll
              for (int j = 0; j < kChunk; ++j) *reinterpret_cast<uint4 *>(o + j * NT * kN) = q[j];
            } else {
#pragma unroll
              for (int j = 0; j < kChunk; ++j) {
                const int w = w0 + j * NT;
                if (vec && w >= cur.lo && w < cur.hi)
                  *reinterpret_cast<uint4 *>(o + j * NT * kN) = q[j];
                else if (w < cur.n)
                  cur.store_ragged(w, q[j], out);
              }
            }
          }
          if (more) nxt.load(s, cps, buf);
        }
      }
      cur = nxt;
    }
    __syncthreads();
  }
  if (C > 1) cluster_sync_all();  // others may still read this CTA's slip
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// The device that holds every given array (NULL ones are skipped): a call
// may name memory of another device than the current one, and a host
// pointer is refused instead of faulting the kernel.  Negative on error.
int device_of(const char *who, std::initializer_list<std::pair<const char *, const void *>> ptrs) {
  int dev = -1;
  for (const auto &p : ptrs) {
    if (!p.second) continue;
    cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p.second);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("%s: %s: %s", who, p.first, cudaGetErrorString(e));
      return -4;
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
      set_error("%s: %s is not device memory", who, p.first);
      return -2;
    }
    if (at.type == cudaMemoryTypeManaged) continue;
    if (dev >= 0 && at.device != dev) {
      set_error("%s: %s is on device %d, other arrays on device %d", who, p.first, at.device, dev);
      return -2;
    }
    dev = at.device;
  }
  if (dev < 0 && cudaGetDevice(&dev) != cudaSuccess) {
    set_error("%s: %s", who, cudaGetErrorString(cudaGetLastError()));
    return -4;
  }
  return dev;
}

int elem_size(int dtype) { return dtype == SNAI_DTYPE_FP32 ? 4 : 2; }

bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Ids and floats are read and written by fours of bytes: an odd address is an
// error here instead of one of the GPU's.  (Host arrays may lie anywhere.)
int check_words(const char *who, std::initializer_list<std::pair<const char *, const void *>> ptrs) {
  for (const auto &p : ptrs)
    if (!aligned(p.second, 4)) {
      set_error("%s: %s is not aligned to 4 bytes", who, p.first);
      return -2;
    }
  return 0;
}

// What every call of this file checks of its rows and temperature.
int check_rows(const char *who, const void *logits, int dtype, int rows, int vocab, long long ld, double t) {
  if (dtype != SNAI_DTYPE_FP32 && dtype != SNAI_DTYPE_BF16 && dtype != SNAI_DTYPE_FP16) {
    set_error("%s: unknown dtype %d", who, dtype);
    return -2;
  }
  if (rows < 0 || rows > kMaxRows) {
    set_error("%s: rows %d outside [0, %d]", who, rows, kMaxRows);
    return -2;
  }
  if (vocab < 1 || vocab > kMaxVocab) {
    set_error("%s: vocab %d outside [1, %d]", who, vocab, kMaxVocab);
    return -2;
  }
  if (ld < vocab || ld > kMaxElems / std::max(rows, 1)) {
    set_error("%s: row stride %lld < vocab %d, or %d such rows beyond any memory", who, ld, vocab, rows);
    return -2;
  }
  if (!(t >= 1e-3 && t <= 1e3)) {
    set_error("%s: temperature %g outside [0.001, 1000]", who, t);
    return -2;
  }
  if (rows > 0 && !logits) {
    set_error("%s: logits is NULL", who);
    return -2;
  }
  if (!aligned(logits, elem_size(dtype))) {
    set_error("%s: logits is not aligned to its elements", who);
    return -2;
  }
  return 0;
}

// The gradient may be the logits' own memory, row for row, or memory that
// shares no element with them (another array, or other columns of rows of
// the same stride).
int check_grad(const char *who, const void *logits, int dtype, int rows, int vocab, long long ld, const void *grad,
               long long gld) {
  if (gld < vocab || gld > kMaxElems / std::max(rows, 1)) {
    set_error("%s: gradient row stride %lld < vocab %d, or %d such rows beyond any memory", who, gld, vocab, rows);
    return -2;
  }
  const long long es = elem_size(dtype);
  if (!aligned(grad, es)) {
    set_error("%s: the gradient is not aligned to its elements", who);
    return -2;
  }
  const intptr_t a = reinterpret_cast<intptr_t>(logits), b = reinterpret_cast<intptr_t>(grad);
  const intptr_t ea = a + ((rows - 1) * ld + vocab) * es, eb = b + ((rows - 1) * gld + vocab) * es;
  if (rows == 0 || a >= eb || b >= ea) return 0;
  if (ld == gld) {
    if (a == b) return 0;
    const intptr_t off = (b > a ? b - a : a - b), pitch = ld * es, in = off % pitch;
    if (in >= vocab * es && pitch - in >= vocab * es) return 0;
  }
  set_error("%s: the gradient overlaps the logits without being the same rows", who);
  return -2;
}

// How rows are cut and spread.
struct Plan {
  int wps, C, nt;
  bool even;
};

// What one row takes in 16-byte words, at most.
int row_words(const void *logits, int dtype, int vocab, long long ld) {
  const int es = elem_size(dtype), kn = 16 / es;
  const int pad = ld * es % 16 == 0 ? (int)((reinterpret_cast<uintptr_t>(logits) & 15) / es) : kn - 1;
  return (pad + vocab + kn - 1) / kn;
}

// Streamed rows: a CTA a row, whatever its length.  When the rows leave SMs
// short of CTAs a row is spread over a cluster of up to 8, down to slices of
// 8 KB, until all CTAs are so many halves of the SMs.
//  7 without alternatives: 131072 fp32, 250 rows 25 us over pairs and 33 over
//    one; past it 400 rows 39 over one and 35 over pairs, but 520 rows of 50001
//    bf16 15 and 16.  (11 would give 150 rows of 131072 17 us over fours for 21
//    over pairs, and 100 rows of 16384 6.1 over eights for 4.7 over fours.)
// 11 with few: 20 of 131072, 200 rows 34 us over fours and 40 over pairs, 250
//    rows 51 and 42, 400 rows 49 over pairs and 62 over one; 512 rows of 16384
//    18.7 over pairs and 17.9 over one.
//  4 with more, whose CTAs are twice as large and merge more: 128 of 131072,
//    100 rows 34 us over pairs and 41 over one, 150 rows 56 and 46; 301 rows of
//    50001 fp16 46 and 28.
Plan plan_stream(const void *logits, int dtype, int rows, int vocab, long long ld, int top_k, int sms) {
  const int words = row_words(logits, dtype, vocab, ld);
  Plan p;
  const long long most = (top_k == 0 ? 7 : top_k <= kFewTop ? 11 : 4) * sms / 2;
  p.C = 1;
  while (p.C < 8 && (long long)rows * p.C * 2 <= most && words / (2 * p.C) >= 512) p.C *= 2;
  p.wps = (words + p.C - 1) / p.C;
  p.nt = top_k <= kFewTop ? 128 : 256;
  p.even = ld * elem_size(dtype) % 16 == 0;
  return p;
}

// Staged rows: a slice holds at most 66 KB, so that three CTAs of an SM have
// a row each in flight or in work.  Longer rows go over a cluster of up to 8
// CTAs, then (few can be that long) slices grow to what one CTA can hold,
// then the cluster to 16.  With fewer rows than SMs a row is spread further,
// down to slices of 8 KB.
Plan plan_staged(const void *logits, int dtype, int rows, int vocab, long long ld, size_t extra, int sms) {
  const int words = row_words(logits, dtype, vocab, ld);
  const size_t bytes = (size_t)words * 16, best = 66 * 1024, most = 224 * 1024 - extra;
  int C = (int)std::min<size_t>((bytes + best - 1) / best, 8);
  if ((bytes + C - 1) / C > most) C = 16;
  while (C <= 4 && (long long)rows * C * 2 <= sms && bytes / (2 * C) >= 8192) C *= 2;
  Plan p;
  p.C = C;
  p.wps = (words + C - 1) / C;
  p.nt = p.wps <= 1024 ? 128 : 256;
  p.even = ld * elem_size(dtype) % 16 == 0;
  return p;
}

// Launches `kern` over the rows with as many clusters as fit the GPU at once
// (asked once per kernel, device and shape), or as many as there are rows.
template <class A>
int launch_rows(const char *who, void (*kern)(A), const A &args, int nt, size_t smem, int dev, cudaStream_t stream) {
  const void *fn = reinterpret_cast<const void *>(kern);
  const int C = args.in.C;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)C;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.blockDim = dim3(nt);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = C > 1 ? 1 : 0;
  cfg.gridDim = dim3((unsigned)C);
  static std::mutex mu;
  static std::map<std::tuple<const void *, int, int, int, size_t>, int> fits;
  int fit = 0;
  try {
    std::lock_guard<std::mutex> g(mu);
    int &f = fits[std::make_tuple(fn, dev, C, nt, smem)];
    if (f == 0) {
      bool ok = set_dyn_smem(kern, 227 * 1024);
      ok = ok && cudaFuncSetAttribute(fn, cudaFuncAttributePreferredSharedMemoryCarveout, 100) == cudaSuccess;
      if (C > 8) ok = ok && cudaFuncSetAttribute(fn, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
      if (C > 1) {
        ok = ok && cudaOccupancyMaxActiveClusters(&f, fn, &cfg) == cudaSuccess;
      } else {
        ok = ok && cudaOccupancyMaxActiveBlocksPerMultiprocessor(&f, fn, nt, smem) == cudaSuccess;
        f *= device_sm_count(dev);
      }
      if (!ok || f < 1) {
        f = 0;
        set_error("%s: rows of %d logits do not fit this GPU: %s", who, args.in.V, cudaGetErrorString(cudaGetLastError()));
        return -4;
      }
    }
    fit = f;
  } catch (const std::exception &x) {  // no exception leaves a C entry
    set_error("%s: %s", who, x.what());
    return -3;
  }
  cfg.gridDim = dim3((unsigned)(std::min(args.in.rows, fit) * C));
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args);
  if (e == cudaSuccess) return 0;
  cudaGetLastError();
  set_error("%s launch failed: %s", who, cudaGetErrorString(e));
  return -4;
}

template <class F>
int by_dtype(int dtype, F &&f) {
  if (dtype == SNAI_DTYPE_FP32) return f(float());
  if (dtype == SNAI_DTYPE_BF16) return f(__nv_bfloat16());
  return f(__half());
}

// Chunks in flight a CTA.  One more each leaves a CTA less an SM: 301 rows of
// 50001 fp16 with 128 alternatives 40 us for 28, 2048 x 131072 fp32 without
// 167 for 155; only calls of few CTAs would gain (200 such rows 20.5 for 23,
// 400 of them 35 for 39).
constexpr int kRing128 = 2, kRing256 = 3;

template <typename E, int NT, int D>
int score_nt(const char *who, const ScoreArgs &a, size_t smem, int dev, cudaStream_t st) {
  if (a.top_k) return launch_rows(who, snai_score<E, NT, D, true, true>, a, NT, smem, dev, st);
  if (a.entropy) return launch_rows(who, snai_score<E, NT, D, false, true>, a, NT, smem, dev, st);
  return launch_rows(who, snai_score<E, NT, D, false, false>, a, NT, smem, dev, st);
}

// mode 0: scores' gradient, 1: distillation; extra: as the kernel's EXTRA
template <typename E, int NT>
int grad_nt(const char *who, const RowGradArgs &a, int mode, int extra, int entry, size_t smem, int dev,
            cudaStream_t st) {
  void (*const kern[2][4])(RowGradArgs) = {
      {snai_row_grad<E, NT, 0, 0>, snai_row_grad<E, NT, 0, 1>, nullptr, nullptr},
      {snai_row_grad<E, NT, 1, 0>, snai_row_grad<E, NT, 1, 1>, snai_row_grad<E, NT, 1, 2>, snai_row_grad<E, NT, 1, 3>}};
  return launch_rows(who, kern[mode][extra], a, NT + entry, smem, dev, st);
}

int launch_row_grad(const char *who, RowGradArgs &a, int dtype, int mode, int extra, int dev, cudaStream_t st) {
  const int ne = a.n + (a.labels ? 1 : 0);
  const size_t lists = (size_t)((ne + 3) & ~3) * 10 * 4 + 256 * 4;
  const int entry = ne > 32 ? 64 : 32;  // entry threads
  const Plan p = plan_staged(a.in.logits, dtype, a.in.rows, a.in.V, a.in.ld, lists, device_sm_count(dev));
  a.in.wps = p.wps;
  a.in.C = p.C;
  a.in.even = p.even;
  const size_t smem = (size_t)p.wps * 16 + lists;
  return by_dtype(dtype, [&](auto e) {
    using E = decltype(e);
    return p.nt == 128 ? grad_nt<E, 128>(who, a, mode, extra, entry, smem, dev, st)
                       : grad_nt<E, 256>(who, a, mode, extra, entry, smem, dev, st);
  });
}

}  // namespace

int check_score(const char *who, const ScoreLaunch &s) {
  int rc = check_rows(who, s.logits, s.dtype, s.rows, s.V, s.ld, s.temperature);
  if (rc) return rc;
  if (s.n_tok < 0 || s.n_tok > kMaxList) {
    set_error("%s: n_tok %d outside [0, %d]", who, s.n_tok, kMaxList);
    return -2;
  }
  if (s.top_k < 0 || s.top_k > std::min(kMaxList, s.V)) {
    set_error("%s: top_k %d outside [0, %d]", who, s.top_k, std::min(kMaxList, s.V));
    return -2;
  }
  if (s.n_tok == 0 && s.top_k == 0 && !s.entropy) {
    set_error("%s: nothing to compute (no tokens, no entropy, no alternatives)", who);
    return -2;
  }
  if (s.rows > 0 && s.n_tok > 0 && (!s.tokens || !s.logprob)) {
    set_error("%s: NULL tokens or logprob", who);
    return -2;
  }
  if (s.rows > 0 && s.top_k > 0 && (!s.top_ids || !s.top_logprob)) {
    set_error("%s: NULL top_ids or top_logprob", who);
    return -2;
  }
  return 0;
}

int launch_score(const char *who, const ScoreLaunch &s, cudaStream_t stream) {
  int rc = check_score(who, s);
  if (rc == 0)
    rc = check_words(who, {{"tokens", s.tokens},
                           {"logprob", s.logprob},
                           {"entropy", s.entropy},
                           {"top_ids", s.top_ids},
                           {"top_logprob", s.top_logprob}});
  if (rc) return rc;
  if (s.rows == 0) return 0;
  const bool tok = s.n_tok > 0, top = s.top_k > 0;
  const int dev = device_of(who, {{"logits", s.logits},
                                  {"tokens", tok ? s.tokens : nullptr},
                                  {"logprob", tok ? s.logprob : nullptr},
                                  {"entropy", s.entropy},
                                  {"top_ids", top ? s.top_ids : nullptr},
                                  {"top_logprob", top ? s.top_logprob : nullptr}});
  if (dev < 0) return dev;
  DeviceGuard g(dev);
  ScoreArgs a{};
  a.in = Rows{s.logits, s.ld, s.rows, s.V, 0, 0, false};
  a.tokens = s.tokens;
  a.n_tok = s.n_tok;
  a.c = (float)(1.4426950408889634 / s.temperature);
  const bool ent = s.top_k > 0 || s.entropy;  // W is at hand
  const double inv = ent ? 1.0 / s.temperature : kLn2d * a.c;
  a.two_t = (float)(2.0 * inv);
  a.two_t_lo = (float)(2.0 * inv - a.two_t);
  a.off = ent ? (float)(1.0 / s.temperature / a.c - kLn2d) : 0.f;
  a.top_k = s.top_k;
  a.logprob = s.logprob;
  a.entropy = s.entropy;
  a.top_ids = s.top_ids;
  a.top_logprob = s.top_logprob;
  // The first chunk's bound lets some 1.2 k to 2 k logits through and three
  // times as many of the next three: with room for 10 k the block meets each
  // time the row has grown fourfold, else each time it has doubled.
  a.soft = s.top_k + s.top_k / 2 + 16;
  for (a.cap = 512; a.cap < max_cap(s.top_k <= kFewTop ? 128 : 256) && a.cap < 10 * s.top_k;) a.cap *= 2;
  a.grow = a.cap >= 10 * s.top_k ? 4 : 2;
  const Plan p = plan_stream(s.logits, s.dtype, s.rows, s.V, s.ld, s.top_k, device_sm_count(dev));
  a.in.wps = p.wps;
  a.in.C = p.C;
  a.in.even = p.even;
  const size_t lists = s.top_k ? (size_t)a.cap * 8 * (p.C > 1 ? 2 : 1) : 0;
  const size_t smem = (size_t)(p.nt == 128 ? kRing128 : kRing256) * kChunk * p.nt * 16 + lists;
  return by_dtype(s.dtype, [&](auto e) {
    using E = decltype(e);
    return p.nt == 128 ? score_nt<E, 128, kRing128>(who, a, smem, dev, stream)
                       : score_nt<E, 256, kRing256>(who, a, smem, dev, stream);
  });
}

int check_distill(const char *who, const DistillLaunch &s) {
  int rc = check_rows(who, s.logits, s.dtype, s.rows, s.V, s.ld, s.temperature);
  if (rc) return rc;
  if (s.top_k < 1 || s.top_k > kMaxList) {
    set_error("%s: top_k %d outside [1, %d]", who, s.top_k, kMaxList);
    return -2;
  }
  if (!(s.label_weight >= 0.0 && s.label_weight <= 1.0)) {
    set_error("%s: label_weight %g outside [0, 1]", who, s.label_weight);
    return -2;
  }
  if (s.rest != 0 && s.rest != 1) {
    set_error("%s: rest %d is neither 0 nor 1", who, s.rest);
    return -2;
  }
  if (s.rows > 0 && s.label_weight > 0.0 && !s.labels) {
    set_error("%s: label_weight %g without labels", who, s.label_weight);
    return -2;
  }
  if (s.rows > 0 && (!s.teacher_ids || !s.teacher_logits || !s.loss)) {
    set_error("%s: NULL teacher_ids, teacher_logits or loss", who);
    return -2;
  }
  return s.grad ? check_grad(who, s.logits, s.dtype, s.rows, s.V, s.ld, s.grad, s.grad_ld) : 0;
}

int launch_distill(const char *who, const DistillLaunch &s, cudaStream_t stream) {
  int rc = check_distill(who, s);
  if (rc == 0)
    rc = check_words(who, {{"teacher_ids", s.teacher_ids},
                           {"teacher_logits", s.teacher_logits},
                           {"labels", s.labels},
                           {"row_grad", s.row_grad},
                           {"loss", s.loss}});
  if (rc) return rc;
  if (s.rows == 0) return 0;
  const int *labels = s.label_weight > 0.0 ? s.labels : nullptr;
  const float *row_grad = s.grad ? s.row_grad : nullptr;
  const int dev = device_of(who, {{"logits", s.logits},
                                  {"teacher_ids", s.teacher_ids},
                                  {"teacher_logits", s.teacher_logits},
                                  {"labels", labels},
                                  {"row_grad", row_grad},
                                  {"loss", s.loss},
                                  {"grad", s.grad}});
  if (dev < 0) return dev;
  DeviceGuard g(dev);
  RowGradArgs a{};
  a.in = Rows{s.logits, s.ld, s.rows, s.V, 0, 0, false};
  a.ids = s.teacher_ids;
  a.vals = s.teacher_logits;
  a.n = s.top_k;
  a.c = (float)(1.4426950408889634 / s.temperature);
  a.inv_t = 1.0 / s.temperature;
  a.inv_t_f = (float)a.inv_t;
  a.labels = labels;
  a.row_grad = row_grad;
  a.t = s.temperature;
  a.a = s.label_weight;
  a.rest = s.rest;
  a.loss = s.loss;
  a.grad = s.grad;
  a.grad_ld = s.grad_ld;
  a.inv_t_z = kLn2d * a.c;
  const int extra = !labels || s.temperature == 1.0 ? 0 : s.temperature == 2.0 ? 2 : s.temperature == 4.0 ? 3 : 1;
  a.one_z = kLn2d * (extra == 1 ? (double)kLog2E : a.c * s.temperature);  // the powers are of c's exponents
  return launch_row_grad(who, a, s.dtype, 1, extra, dev, stream);
}

}  // namespace snai

using namespace snai;

extern "C" int cortex_score(const void *logits, int dtype, int rows, int vocab, long long ld, const int *tokens,
                            int n_tok, double temperature, int top_k, float *logprob, float *entropy, int *top_ids,
                            float *top_logprob, void *stream) {
  clear_error();
  ScoreLaunch s;
  s.logits = logits;
  s.dtype = dtype;
  s.rows = rows;
  s.V = vocab;
  s.ld = ld;
  s.tokens = tokens;
  s.n_tok = n_tok;
  s.temperature = temperature;
  s.top_k = top_k;
  s.logprob = logprob;
  s.entropy = entropy;
  s.top_ids = top_ids;
  s.top_logprob = top_logprob;
  return launch_score("cortex_score", s, static_cast<cudaStream_t>(stream));
}

extern "C" int cortex_score_grad(const void *logits, int dtype, int rows, int vocab, long long ld, const int *tokens,
                                 int n_tok, double temperature, const float *g_logprob, const float *g_entropy,
                                 void *grad, long long grad_ld, void *stream) {
  clear_error();
  const char *who = "cortex_score_grad";
  int rc = check_rows(who, logits, dtype, rows, vocab, ld, temperature);
  if (rc) return rc;
  if (n_tok < 0 || n_tok > kMaxList) {
    set_error("%s: n_tok %d outside [0, %d]", who, n_tok, kMaxList);
    return -2;
  }
  if (n_tok == 0 && !g_entropy) {
    set_error("%s: nothing to propagate (no tokens, no g_entropy)", who);
    return -2;
  }
  if (rows > 0 && (!grad || (n_tok > 0 && (!tokens || !g_logprob)))) {
    set_error("%s: NULL grad, tokens or g_logprob", who);
    return -2;
  }
  rc = check_words(who, {{"tokens", tokens}, {"g_logprob", g_logprob}, {"g_entropy", g_entropy}});
  if (rc == 0) rc = check_grad(who, logits, dtype, rows, vocab, ld, grad, grad_ld);
  if (rc) return rc;
  if (rows == 0) return 0;
  if (n_tok == 0) tokens = nullptr, g_logprob = nullptr;
  const int dev = device_of(who, {{"logits", logits},
                                  {"tokens", tokens},
                                  {"g_logprob", g_logprob},
                                  {"g_entropy", g_entropy},
                                  {"grad", grad}});
  if (dev < 0) return dev;
  DeviceGuard g(dev);
  RowGradArgs a{};
  a.in = Rows{logits, ld, rows, vocab, 0, 0, false};
  a.ids = tokens;
  a.vals = g_logprob;
  a.n = n_tok;
  a.c = (float)(1.4426950408889634 / temperature);
  a.inv_t = 1.0 / temperature;
  a.inv_t_f = (float)a.inv_t;
  a.g_entropy = g_entropy;
  a.grad = grad;
  a.grad_ld = grad_ld;
  return launch_row_grad(who, a, dtype, 0, g_entropy ? 1 : 0, dev, static_cast<cudaStream_t>(stream));
}

extern "C" int cortex_distill(const void *logits, int dtype, int rows, int vocab, long long ld,
                              const int *teacher_ids, const float *teacher_logits, int top_k, const int *labels,
                              const float *row_grad, const snai_distill_params *params, float *loss, void *grad,
                              long long grad_ld, void *stream) {
  clear_error();
  if (!params) {
    set_error("cortex_distill: params is NULL");
    return -1;
  }
  DistillLaunch s;
  s.logits = logits;
  s.dtype = dtype;
  s.rows = rows;
  s.V = vocab;
  s.ld = ld;
  s.teacher_ids = teacher_ids;
  s.teacher_logits = teacher_logits;
  s.top_k = top_k;
  s.labels = labels;
  s.row_grad = row_grad;
  s.temperature = params->temperature;
  s.label_weight = params->label_weight;
  s.rest = params->rest;
  s.loss = loss;
  s.grad = grad;
  s.grad_ld = grad_ld;
  return launch_distill("cortex_distill", s, static_cast<cudaStream_t>(stream));
}
