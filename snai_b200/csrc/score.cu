// score.cu - operators over rows of vocabulary logits: log probabilities of
// given tokens with entropy and top alternatives, their gradient, and the
// distillation loss against a teacher's top logits with its gradient
// (cortex_score, cortex_score_grad, cortex_distill in include/cortex.h).
//
// With T the temperature, m the row's maximum, d_i = (z_i - m) / T,
// e_i = exp(d_i) and S = sum e_i:
//   log p_i = d_i - log S,  entropy H = log S - sum(e_i d_i) / S.
// A masked logit (-inf) has e_i = 0 and takes no gradient; a row holding a
// NaN or +inf has no distribution and yields NaN (its alternatives' ids -1).
#include <cuda_fp16.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <initializer_list>
#include <utility>

#include "../../include/cortex.h"
#include "common.cuh"
#include "engine.h"

namespace snai {
namespace {

constexpr int kThreads = 512;
constexpr int kMaxList = kScoreMaxK;
constexpr int kMaxVocab = 1 << 19; // as cortex_sample

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// maximum that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Sort key of a logit and its id: descending value, then ascending id.
__device__ __forceinline__ unsigned long long sort_key(float z, int id) {
  const int b = __float_as_int(z + 0.0f);  // -0 counts as +0
  const unsigned k = (unsigned)b ^ (b < 0 ? 0xffffffffu : 0x80000000u);
  return ((unsigned long long)k << 32) | (unsigned)~id;
}

template <typename F>
__device__ __forceinline__ auto block_reduce(decltype(F::id()) v, decltype(F::id()) *red) {
  for (int o = 16; o > 0; o >>= 1) v = F::op(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < (int)(blockDim.x >> 5); ++w) v = F::op(v, red[w]);
  return v;
}
struct MaxOp {
  __device__ static float id() { return -FLT_MAX; }
  __device__ static float op(float a, float b) { return max_nan(a, b); }
};
struct SumOp {
  __device__ static float id() { return 0.f; }
  __device__ static float op(float a, float b) { return a + b; }
};
struct SumD {
  __device__ static double id() { return 0.0; }
  __device__ static double op(double a, double b) { return a + b; }
};
struct SumI {
  __device__ static int id() { return 0; }
  __device__ static int op(int a, int b) { return a + b; }
};

struct ScoreArgs {
  const void *logits;
  long long ld;
  int rows, V;
  const int *tokens;
  int n_tok;
  float inv_t;
  int top_k;
  float *logprob, *entropy;
  int *top_ids;
  float *top_logprob;
};

template <typename E>
__global__ void __launch_bounds__(kThreads) snai_score(const ScoreArgs a) {
  __shared__ float redf[32];
  __shared__ int redi[32];
  __shared__ unsigned long long cand[kMaxList];
  __shared__ int n_cand;
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const E *z = static_cast<const E *>(a.logits) + (long long)r * a.ld;
    float m = -FLT_MAX;
    for (int i = threadIdx.x; i < a.V; i += kThreads) m = max_nan(m, to_f(z[i]));
    m = block_reduce<MaxOp>(m, redf);
    float s = 0.f, w = 0.f;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const float d = max_nan((to_f(z[i]) - m) * a.inv_t, -150.f), e = __expf(d);
      s += e;
      w += e * d;
    }
    s = block_reduce<SumOp>(s, redf);
    w = block_reduce<SumOp>(w, redf);
    const bool bad = !(s < INFINITY);
    const float ls = logf(s);
    for (int j = threadIdx.x; j < a.n_tok; j += kThreads) {
      const int t = a.tokens[(long long)r * a.n_tok + j];
      a.logprob[(long long)r * a.n_tok + j] =
          t < 0 || t >= a.V ? 0.f : bad ? NAN : s == 0.f ? -INFINITY : (to_f(z[t]) - m) * a.inv_t - ls;
    }
    if (threadIdx.x == 0 && a.entropy) a.entropy[r] = bad ? NAN : s == 0.f ? 0.f : ls - w / s;
    if (!a.top_k) continue;
    int *ids = a.top_ids + (long long)r * a.top_k;
    float *lps = a.top_logprob + (long long)r * a.top_k;
    if (bad) {
      for (int j = threadIdx.x; j < a.top_k; j += kThreads) ids[j] = -1, lps[j] = NAN;
      continue;
    }
    // the k-th largest key by bisection over the 64-bit keys
    unsigned long long lo = 0, hi = ~0ull;  // count(>= lo) >= k
    while (lo < hi) {
      const unsigned long long mid = lo + (hi - lo) / 2 + 1;
      int c = 0;
      for (int i = threadIdx.x; i < a.V; i += kThreads) c += sort_key(to_f(z[i]), i) >= mid;
      if (block_reduce<SumI>(c, redi) >= a.top_k)
        lo = mid;
      else
        hi = mid - 1;
    }
    if (threadIdx.x == 0) n_cand = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const unsigned long long k = sort_key(to_f(z[i]), i);
      if (k >= lo) cand[atomicAdd(&n_cand, 1)] = k;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < a.top_k; j += kThreads) {
      int rank = 0;
      for (int l = 0; l < a.top_k; ++l) rank += cand[l] > cand[j];
      const int id = (int)~(unsigned)cand[j];
      ids[rank] = id;
      lps[rank] = s == 0.f ? -INFINITY : (to_f(z[id]) - m) * a.inv_t - ls;
    }
    __syncthreads();
  }
}

struct RowGradArgs {
  const void *logits;
  long long ld;
  int rows, V;
  const int *ids;  // [rows][n] tokens or teacher ids
  int n;
  const float *vals;  // [rows][n] g_logprob or teacher logits
  float inv_t;
  double inv_td;
  const float *g_entropy;
  const int *labels;
  const float *row_grad;
  float t, t2, a;  // temperature, temperature^2, label weight
  int rest;
  float *loss;
  void *grad;
  long long grad_ld;
};

// MODE 0: the gradient of scores; MODE 1: distillation.
template <typename E, int MODE>
__global__ void __launch_bounds__(kThreads) snai_row_grad(const RowGradArgs a) {
  __shared__ float redf[32];
  __shared__ double redd[32];
  __shared__ int redi[32];
  __shared__ int ids[kMaxList];
  __shared__ double q[kMaxList];   // weights (MODE 0: g)
  __shared__ double lq[kMaxList];
  for (int r = blockIdx.x; r < a.rows; r += gridDim.x) {
    const E *z = static_cast<const E *>(a.logits) + (long long)r * a.ld;
    E *gr = a.grad ? static_cast<E *>(a.grad) + (long long)r * a.grad_ld : nullptr;
    int valid = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < a.n; j += kThreads) {
      const int id = a.ids[(long long)r * a.n + j];
      const bool in = id >= 0 && id < a.V;
      ids[j] = in ? id : -1;
      valid += in;
      q[j] = in ? (double)a.vals[(long long)r * a.n + j] : 0.0;
    }
    valid = block_reduce<SumI>(valid, redi);
    const int y = MODE == 1 && a.labels && a.labels[r] >= 0 && a.labels[r] < a.V ? a.labels[r] : -1;
    const float gh = MODE == 0 && a.g_entropy ? a.g_entropy[r] : 0.f;
    if (!valid && y < 0 && gh == 0.f) {  // a row of padding
      if (MODE == 1 && threadIdx.x == 0) a.loss[r] = 0.f;
      if (gr)
        for (int i = threadIdx.x; i < a.V; i += kThreads) gr[i] = from_f<E>(0.f);
      continue;
    }
    float m = -FLT_MAX;
    for (int i = threadIdx.x; i < a.V; i += kThreads) m = max_nan(m, to_f(z[i]));
    m = block_reduce<MaxOp>(m, redf);
    auto listed = [&](int i) {
      for (int j = 0; j < a.n; ++j)
        if (ids[j] == i) return true;
      return false;
    };
    float s = 0.f, w = 0.f, s1 = 0.f, u = 0.f;
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const float zi = to_f(z[i]), d = max_nan((zi - m) * a.inv_t, -150.f), e = __expf(d);
      s += e;
      w += e * d;
      if (MODE == 1) s1 += __expf(max_nan(zi - m, -150.f));
      if (MODE == 1 && a.rest && !listed(i)) u += e;
    }
    s = block_reduce<SumOp>(s, redf);
    w = block_reduce<SumOp>(w, redf);
    s1 = block_reduce<SumOp>(s1, redf);
    u = block_reduce<SumOp>(u, redf);
    const float ls = logf(s), inv_s = s > 0.f ? 1.f / s : s == 0.f ? 0.f : NAN;
    float gsum = 0.f, cr = 0.f, mass = 0.f;
    const float wy = y >= 0 ? a.a : 0.f;
    if (MODE == 0) {
      float g = 0.f;
      for (int j = threadIdx.x; j < a.n; j += kThreads) g += (float)q[j];
      gsum = block_reduce<SumOp>(g, redf);
    } else {
      double tm = -INFINITY;
      for (int j = 0; j < a.n; ++j)
        if (ids[j] >= 0) tm = fmax(tm, q[j]);
      if (tm == -INFINITY) tm = 0;  // a list without mass
      double ts = 0;
      for (int j = threadIdx.x; j < a.n; j += kThreads)
        if (ids[j] >= 0) ts += exp((q[j] - tm) * a.inv_td);
      ts = block_reduce<SumD>(ts, redd);
      double kl = 0, qs = 0;
      for (int j = threadIdx.x; j < a.n; j += kThreads) {
        lq[j] = a.rest ? q[j] : (q[j] - tm) * a.inv_td - log(ts);
        const double qj = ids[j] >= 0 && q[j] != -INFINITY ? exp(lq[j]) : 0.0;
        q[j] = qj;
        if (qj > 0) {
          const double zj = to_f(z[ids[j]]);
          kl += qj * (lq[j] - (zj == -INFINITY ? zj : (zj - m) * a.inv_td - log((double)s)));
        }
        qs += qj;
      }
      kl = block_reduce<SumD>(kl, redd);
      qs = block_reduce<SumD>(qs, redd);
      double rr = 0;
      if (a.rest && valid && u > 0.f) {
        rr = fmax(0.0, 1.0 - qs);
        if (rr > 0) kl += rr * (log(rr) - log((double)u / s));
        cr = (float)(rr / u);
      }
      mass = (float)(qs + rr);
      if (threadIdx.x == 0) {
        double l = a.a < 1.f ? (1.0 - a.a) * a.t2 * kl : 0.0;
        const double zy = y >= 0 ? to_f(z[y]) : 0.f;
        if (y >= 0) l -= a.a * (zy == -INFINITY ? zy : zy - m - log((double)s1));
        a.loss[r] = inv_s != inv_s ? NAN : (float)l;
      }
    }
    if (!gr) continue;
    const float rg = MODE == 1 && a.row_grad ? a.row_grad[r] : 1.f;
    __syncthreads();
    for (int i = threadIdx.x; i < a.V; i += kThreads) {
      const float zi = to_f(z[i]), d = max_nan((zi - m) * a.inv_t, -150.f), e = __expf(d);
      float g = 0.f;
      if (MODE == 0) {
        float hot = 0.f;
        for (int j = 0; j < a.n; ++j)
          if (ids[j] == i) hot += (float)q[j];
        const float p = e * inv_s;
        g = (hot - p * gsum - gh * p * (d - w * inv_s)) * a.inv_t;
      } else {
        double hot = 0;
        bool on = false;
        for (int j = 0; j < a.n; ++j)
          if (ids[j] == i) hot += q[j], on = true;
        g = (1.f - a.a) * a.t * (e * mass * inv_s - (float)hot - (on ? 0.f : e * cr));
        if (y >= 0) g += wy * (__expf(max_nan(zi - m, -150.f)) / s1 - (i == y ? 1.f : 0.f));
        g *= rg;
      }
      gr[i] = from_f<E>(zi == -INFINITY ? (inv_s != inv_s ? NAN : 0.f) : inv_s != inv_s ? NAN : g);
    }
  }
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

// What every call of this file checks of its rows and temperature.
int check_rows(const char *who, const void *logits, int dtype, int rows, int vocab, long long ld, double t) {
  if (dtype != SNAI_DTYPE_FP32 && dtype != SNAI_DTYPE_BF16 && dtype != SNAI_DTYPE_FP16) {
    set_error("%s: unknown dtype %d", who, dtype);
    return -2;
  }
  if (rows < 0) {
    set_error("%s: rows < 0", who);
    return -2;
  }
  if (vocab < 1 || vocab > kMaxVocab) {
    set_error("%s: vocab %d outside [1, %d]", who, vocab, kMaxVocab);
    return -2;
  }
  if (ld < vocab || ld > (1ll << 40)) {
    set_error("%s: row stride %lld < vocab %d", who, ld, vocab);
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
  if (gld < vocab || gld > (1ll << 40)) {
    set_error("%s: gradient row stride %lld < vocab %d", who, gld, vocab);
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

int launched(const char *who) {
  const cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess) return 0;
  set_error("%s launch failed: %s", who, cudaGetErrorString(e));
  return -4;
}

template <class F>
void by_dtype(int dtype, F &&f) {
  if (dtype == SNAI_DTYPE_FP32)
    f(float());
  else if (dtype == SNAI_DTYPE_BF16)
    f(__nv_bfloat16());
  else
    f(__half());
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
  const int rc = check_score(who, s);
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
  const ScoreArgs a{s.logits,  s.ld,    s.rows,      s.V,       s.tokens,   s.n_tok, (float)(1.0 / s.temperature),
                    s.top_k,   s.logprob, s.entropy, s.top_ids, s.top_logprob};
  const int grid = std::min(s.rows, 4 * device_sm_count(dev));
  by_dtype(s.dtype, [&](auto e) { snai_score<decltype(e)><<<grid, kThreads, 0, stream>>>(a); });
  return launched(who);
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
  const int rc = check_distill(who, s);
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
  a.logits = s.logits, a.ld = s.ld, a.rows = s.rows, a.V = s.V;
  a.ids = s.teacher_ids, a.n = s.top_k, a.vals = s.teacher_logits, a.labels = labels, a.row_grad = row_grad;
  a.inv_td = 1.0 / s.temperature, a.inv_t = (float)a.inv_td;
  a.t = (float)s.temperature, a.t2 = (float)(s.temperature * s.temperature);
  a.a = (float)s.label_weight, a.rest = s.rest;
  a.loss = s.loss, a.grad = s.grad, a.grad_ld = s.grad_ld;
  const int grid = std::min(s.rows, 4 * device_sm_count(dev));
  by_dtype(s.dtype, [&](auto e) { snai_row_grad<decltype(e), 1><<<grid, kThreads, 0, stream>>>(a); });
  return launched(who);
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
  rc = check_grad(who, logits, dtype, rows, vocab, ld, grad, grad_ld);
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
  a.logits = logits, a.ld = ld, a.rows = rows, a.V = vocab;
  a.ids = tokens, a.n = n_tok, a.vals = g_logprob, a.g_entropy = g_entropy;
  a.inv_td = 1.0 / temperature, a.inv_t = (float)a.inv_td;
  a.grad = grad, a.grad_ld = grad_ld;
  const int grid = std::min(rows, 4 * device_sm_count(dev));
  by_dtype(dtype, [&](auto e) {
    snai_row_grad<decltype(e), 0><<<grid, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  });
  return launched(who);
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
