// Log probabilities of given tokens, the entropy of their distributions and the likeliest alternatives, from logits
// [rows, V], and the gradient of the first two and of the normaliser.  With u = l / T:
//   lse = log sum exp(u),  logp = u[t] - lse,  H = lse - sum p u,  p = exp(u - lse)
//   dl  = 1/T (dlogp (delta_t - p) + dlse p - dH p (log p + H))
//
// Forward is one pass with a running maximum: a thread holds (m, S, D) = (max l, sum e, sum (l - m) e), e = exp((l - m) / T),
// and two such triples over different elements join by rescaling the one with the smaller m.  Then lse = m / T + log S and
// H = log S - D / (T S): differences from the maximum, so that nothing large cancels.
//
// Alternatives: a second pass over the row, which the caches still hold, collects the elements that are at least a bound
// with no fewer than k of them above it, some tens in all, and one wave sorts those.  The order is by value and then the
// lower index, so ties have one answer.
//
// Bound: HBM; forward reads the logits once, backward reads them and writes their gradient.
#include "row_vec.h"
#include "topk_wave.h"

namespace maba {
namespace logprobs {

using namespace rowvec;

constexpr float LOWEST = -3.40282347e38f, LOG2E = 1.4426950408889634f;

struct Logits {
  const char* p;
  int64_t outer, inner, per;        // bytes from row to row, `per` rows of one outer step
  __device__ __forceinline__ const char* row(int64_t r) const { return p + (r / per) * outer + (r % per) * inner; }
};

struct ForwardArgs {
  Logits x;
  const int64_t* targets;
  float *logp, *entropy, *lse, *top_logp;
  int64_t* top_ids;
  int64_t R;
  int V, k;
  float inv;                         // 1 / T
};

// The order of alternatives: by value (NaN above all, -0 as +0), then the lower index.
__device__ __forceinline__ key64 order_key(float v, uint32_t idx) {
  const uint32_t o = v != v ? 0xffffffffu : order_f32(v + 0.f);
  return ((key64)o << 32) | (key64)(~idx);
}

struct Triple { float m, s, d; };
// D of a state whose maximum rises by -dm, f = exp2(dm c).  dm may be past fp32's range, and f is zero then.
__device__ __forceinline__ float moved(float d, float s, float dm, float f) { return d * f + fmaxf(dm, LOWEST) * f * s; }
// Joined; a triple of no mass takes no part, whatever its maximum.
__device__ __forceinline__ Triple join(Triple a, Triple b, float c) {
  const float m = fmaxf(a.m, b.m), da = a.m - m, db = b.m - m;
  const float fa = __builtin_amdgcn_exp2f(da * c), fb = __builtin_amdgcn_exp2f(db * c);
  Triple r = {m, 0.f, 0.f};
  if (a.s != 0.f) { r.s += a.s * fa; r.d += moved(a.d, a.s, da, fa); }
  if (b.s != 0.f) { r.s += b.s * fb; r.d += moved(b.d, b.s, db, fb); }
  return r;
}

// The running state of a thread over its elements, and the largest of them.
template <bool TOP>
struct Running {
  Triple t = {LOWEST, 0.f, 0.f};
  float best = -INFINITY;
  uint32_t best_idx = 0;
  bool any = false;
  // N elements, in the order of their indexes: element e has index idx(e)
  template <int N, class Idx>
  __device__ __forceinline__ void take(const float (&v)[N], float c, Idx idx) {
    float b = v[0];
#pragma unroll
    for (int e = 1; e < N; ++e) b = fmaxf(b, v[e]);
    const float m = fmaxf(t.m, b), dm = t.m - m, f = __builtin_amdgcn_exp2f(dm * c);
    float s = t.s * f, d = moved(t.d, t.s, dm, f);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = v[e] - m, p = __builtin_amdgcn_exp2f(x * c);
      s += p;
      d = fmaf(fmaxf(x, LOWEST), p, d);          // -inf times a p of zero is zero here
    }
    t = {m, s, d};
    if (TOP && b > best) {
      best = b;
      any = true;
#pragma unroll
      for (int e = N - 1; e >= 0; --e)
        if (v[e] == b) best_idx = idx(e);
    }
  }
};

// f(chunk values, first index) over the row's chunks of a group of `lanes` threads, NB at a time while all are whole
template <class T, int NB, class F>
__device__ __forceinline__ void for_chunks(const char* row, int V, int lane, int lanes, F f) {
  constexpr int E = Traits<T>::VEC;
  const int whole = V / E, rounds = whole / (lanes * NB);
  for (int i = 0; i < rounds; ++i) {
    u32x4 u[NB];
    const int c0 = i * lanes * NB + lane;
#pragma unroll
    for (int b = 0; b < NB; ++b) u[b] = load_chunk<T>(row, (uint32_t)(c0 + b * lanes) * 16u, E);
    float v[NB * E];
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      float w[E];
      unpack<T>(u[b], w);
#pragma unroll
      for (int e = 0; e < E; ++e) v[b * E + e] = w[e];
    }
    f(v, c0 * E);
  }
  for (int c = rounds * lanes * NB + lane; c * E < V; c += lanes) {
    float w[E];
    const int left = V - c * E;
    unpack<T>(load_chunk<T>(row, (uint32_t)c * 16u, left), w);
#pragma unroll
    for (int e = 0; e < E; ++e) w[e] = e < left ? w[e] : -INFINITY;
    f(w, c * E);
  }
}

// W waves a row.  One wave for short rows, four of them in a workgroup; otherwise the workgroup is one row's.
template <class T, int W, bool TOP>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void logprobs_kernel(ForwardArgs a) {
  constexpr int E = Traits<T>::VEC, NB = 32 / E, LANES = 64 * W, GROUPS = W == 1 ? 4 : 1, CAP = W == 1 ? 512 : 2048;
  __shared__ Triple s_t[GROUPS * W];
  __shared__ key64 s_max[W], s_min[W], s_found[TOP ? GROUPS * CAP : 1];
  __shared__ int s_count[GROUPS];
  const int group = W == 1 ? threadIdx.x >> 6 : 0, lane = threadIdx.x & (LANES - 1), wave = W == 1 ? 0 : threadIdx.x >> 6;
  const int64_t r = (int64_t)blockIdx.x * GROUPS + __builtin_amdgcn_readfirstlane(group);
  if (W == 1 && r >= a.R) return;               // nothing below waits for another wave where W is 1
  const char* row = a.x.row(r);
  const float c = a.inv * LOG2E;
  const int64_t target = a.targets[r];
  float lt = 0.f;
  if (target >= 0 && target < a.V) {
    float w[E];
    unpack<T>(load_chunk<T>(row + target * (16 / E), 0, 1), w);
    lt = w[0];
  }
  Running<TOP> run;
  for_chunks<T, NB>(row, a.V, lane, LANES, [&](auto& v, int first) {
    run.take(v, c, [&](int e) { return (uint32_t)(first + (e / E) * LANES * E + e % E); });
  });
  Triple t = run.t;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1)
    t = join(t, {__shfl_xor(t.m, off), __shfl_xor(t.s, off), __shfl_xor(t.d, off)}, c);
  key64 bound = KEY_NONE;
  if constexpr (TOP) {
    // Of a wave's lanes' maxima, sorted: the k-th of any wave has k elements above it, and so has the smallest of all
    // waves' (k / W)-th.
    const key64 sorted = wave_sort_desc(run.any ? order_key(run.best, run.best_idx) : KEY_NONE);
    const key64 kth = __shfl(sorted, a.k - 1), part = __shfl(sorted, (a.k + W - 1) / W - 1);
    if constexpr (W == 1) {
      bound = kth;
    } else if ((threadIdx.x & 63) == 0) {
      s_max[wave] = kth;
      s_min[wave] = part;
    }
    if (lane == 0) s_count[group] = 0;
  }
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) s_t[wave] = t;
    __syncthreads();
    t = s_t[0];
#pragma unroll
    for (int w = 1; w < W; ++w) t = join(t, s_t[w], c);
    if constexpr (TOP) {
      key64 lo = s_min[0];
      bound = s_max[0];
#pragma unroll
      for (int w = 1; w < W; ++w) {
        bound = kmax(bound, s_max[w]);
        lo = kmin(lo, s_min[w]);
      }
      bound = kmax(bound, lo);
    }
  }
  const float log_s = logf(t.s), lse = fmaf(t.m, a.inv, log_s);
  const bool none = lse == -INFINITY;            // every logit is -inf: so are the log probabilities, and the entropy is 0
  if (lane == 0) {
    a.lse[r] = lse;
    a.entropy[r] = none ? 0.f : log_s - a.inv * (t.d / t.s);
    a.logp[r] = target < 0 ? 0.f : target >= a.V ? NAN : none ? -INFINITY : (lt - t.m) * a.inv - log_s;
  }
  if constexpr (TOP) {
    const float at_least = bound == KEY_NONE ? -INFINITY : key_score(bound);
    key64* found = s_found + group * CAP;
    const auto collect = [&](auto put) {
      for_chunks<T, NB>(row, a.V, lane, LANES, [&](auto& v, int first) {
        constexpr int N = sizeof(v) / sizeof(v[0]);
        bool any = false;
#pragma unroll
        for (int e = 0; e < N; ++e) any |= !(v[e] < at_least);
        if (!__any(any)) return;
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const int idx = first + (e / E) * LANES * E + e % E;
          const key64 key = order_key(v[e], (uint32_t)idx);
          const bool in = idx < a.V && key >= bound;
          if (__any(in)) put(in ? key : KEY_NONE);
        }
      });
    };
    collect([&](key64 key) {
      if (key != KEY_NONE) {
        const int at = atomicAdd(&s_count[group], 1);
        if (at < CAP) found[at] = key;
      }
    });
    if constexpr (W > 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (wave != 0) return;
    const int l = threadIdx.x & 63, n = *(volatile int*)&s_count[group];
    key64 list = KEY_NONE;
    if (n <= CAP) {
      for (int i = 0; i < n; i += 64) list = wave_merge_topk(list, i + l < n ? found[i + l] : KEY_NONE, 64);
    } else {
      // More than the buffer holds (thousands of the same lanes' elements above the rest): wave 0 goes over the row alone.
      for (int i = 0; i < a.V; i += 64) {
        float w[E];
        key64 key = KEY_NONE;
        if (i + l < a.V) {
          unpack<T>(load_chunk<T>(row + (int64_t)(i + l) * (16 / E), 0, 1), w);
          key = order_key(w[0], (uint32_t)(i + l));
        }
        list = wave_merge_topk(list, key, a.k);
      }
    }
    if (l < a.k) {
      const uint32_t idx = key_index(list);
      float w[E];
      unpack<T>(load_chunk<T>(row + (int64_t)idx * (16 / E), 0, 1), w);
      a.top_ids[r * a.k + l] = (int64_t)idx;
      a.top_logp[r * a.k + l] = none ? -INFINITY : (w[0] - t.m) * a.inv - log_s;
    }
  }
}

struct BackwardArgs {
  Logits x, dx;
  const int64_t* targets;
  const float *dlogp, *dentropy, *dlse, *lse, *entropy;
  int64_t R;
  int V, lg, parts;                  // 2^lg threads a row and `parts` workgroups side by side on it
  float inv;
};

template <class T>
__global__ __launch_bounds__(256) void logprobs_back_kernel(BackwardArgs a) {
  constexpr int E = Traits<T>::VEC, NB = 2;
  const int64_t r = (int64_t)blockIdx.x / a.parts * (256 >> a.lg) + __builtin_amdgcn_readfirstlane(threadIdx.x >> a.lg);
  if (r >= a.R) return;
  const char* row = a.x.row(r);
  char* out = (char*)a.dx.row(r);
  const int64_t target = a.targets[r];
  float lse = a.lse[r];
  const float h = a.entropy[r], gh = a.dentropy ? a.dentropy[r] : 0.f;
  float gl = target < 0 || !a.dlogp ? 0.f : target >= a.V ? NAN : a.dlogp[r], gz = a.dlse ? a.dlse[r] : 0.f;
  if (lse == -INFINITY) {            // no mass: no element has a gradient
    lse = -LOWEST;
    gl = 0.f;
  }
  const float base = gz - gl - (gh != 0.f ? gh * h : 0.f), at_target = gl * a.inv;
  const int lanes = a.parts << a.lg, lane = ((int)(blockIdx.x % a.parts) << a.lg) + (threadIdx.x & ((1 << a.lg) - 1));
  const int mine = target >= 0 && target < a.V ? (int)(target / E) : -1, chunks = (a.V + E - 1) / E;
  for (int c0 = lane; c0 < chunks; c0 += lanes * NB) {
    u32x4 u[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) u[b] = load_chunk<T>(row, (uint32_t)(c0 + b * lanes) * 16u, a.V - (c0 + b * lanes) * E);
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int ch = c0 + b * lanes;
      float v[E];
      unpack<T>(u[b], v);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float lp = fmaf(v[e], a.inv, -lse), p = __builtin_amdgcn_exp2f(lp * LOG2E);
        // where p is zero log p may be -inf: bounded, its product with p is zero
        v[e] = a.inv * p * fmaf(-gh, fmaxf(lp, -1e4f), base);
      }
      if (ch == mine)
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += e == (int)(target % E) ? at_target : 0.f;
      store_chunk<T>(out, (uint32_t)ch * 16u, a.V - ch * E, pack<T>(v));
    }
  }
}

// ---------------------------------------------------------------- arguments

static int check_logits(const maba_tensor* t, const char* who, const char* name, int64_t& rows) {
  if (!t) return fail(MABA_ERR_INVALID, "%s: %s is missing", who, name);
  if (t->ndim != 2 && t->ndim != 3) return fail(MABA_ERR_INVALID, "%s: %s must be [M,V] or [B,L,V], got %dD", who, name, t->ndim);
  if (!is_float_dt(t->dtype)) return fail(MABA_ERR_DTYPE, "%s: f32, f16 or bf16 only, got dtype code %d", who, t->dtype);
  const int n = t->ndim;
  if (t->shape[n - 1] < 1) return fail(MABA_ERR_INVALID, "%s: the vocabulary must not be empty", who);
  if (t->shape[n - 1] > (1 << 28)) return fail(MABA_ERR_UNSUPPORTED, "%s: at most %d tokens", who, 1 << 28);
  if (t->shape[n - 1] > 1 && t->stride[n - 1] != 1) return fail(MABA_ERR_INVALID, "%s: %s needs unit column stride", who, name);
  rows = t->shape[0] * (n == 3 ? t->shape[1] : 1);
  for (int i = 0; i < n; ++i)
    if (t->stride[i] < 0) return fail(MABA_ERR_INVALID, "%s: %s has a negative stride", who, name);
  if (rows > 0x7fffffff) return fail(MABA_ERR_UNSUPPORTED, "%s: too many rows", who);
  if (rows > 0 && !t->data) return fail(MABA_ERR_INVALID, "%s: %s has no data", who, name);
  return MABA_OK;
}
static int check_row_vec(const maba_tensor* t, const char* who, const char* name, int dtype, int64_t rows) {
  if (!t) return fail(MABA_ERR_INVALID, "%s: %s is missing", who, name);
  if (t->dtype != dtype) return fail(MABA_ERR_DTYPE, "%s: %s has dtype code %d, expected %d", who, name, t->dtype, dtype);
  if (t->ndim != 1 || t->shape[0] != rows || (rows > 1 && t->stride[0] != 1))
    return fail(MABA_ERR_INVALID, "%s: %s must be contiguous [%lld]", who, name, (long long)rows);
  if (rows > 0 && !t->data) return fail(MABA_ERR_INVALID, "%s: %s has no data", who, name);
  return MABA_OK;
}
static Logits logits_of(const maba_tensor* t) {
  const int64_t size = t->dtype == MABA_F32 ? 4 : 2;
  if (t->ndim == 2) return {(const char*)t->data, 0, t->stride[0] * size, std::max<int64_t>(t->shape[0], 1)};
  return {(const char*)t->data, t->stride[0] * size, t->stride[1] * size, std::max<int64_t>(t->shape[1], 1)};
}

}  // namespace logprobs
}  // namespace maba

using namespace maba;
using namespace maba::logprobs;
using ffn::overlap;

extern "C" int maba_hip_token_logprobs(const maba_tensor* logits, const maba_tensor* targets, double temperature,
                                       maba_tensor* logp, maba_tensor* entropy, maba_tensor* lse, maba_tensor* top_logp,
                                       maba_tensor* top_ids, void* stream) {
  const char* who = "token_logprobs";
  int64_t R = 0;
  int rc = check_logits(logits, who, "logits", R);
  if (!rc && !(temperature > 0.0 && 1.0 / temperature <= 1e30 && 1.0 / temperature >= 1e-30))
    rc = fail(MABA_ERR_INVALID, "%s: temperature=%g must be positive", who, temperature);
  if (!rc) rc = check_row_vec(targets, who, "targets", MABA_I64, R);
  if (!rc) rc = check_row_vec(logp, who, "logp", MABA_F32, R);
  if (!rc) rc = check_row_vec(entropy, who, "entropy", MABA_F32, R);
  if (!rc) rc = check_row_vec(lse, who, "lse", MABA_F32, R);
  if (rc) return rc;
  const int64_t V = logits->shape[logits->ndim - 1];
  int64_t k = 0;
  if (!top_logp != !top_ids) return fail(MABA_ERR_INVALID, "%s: top_logp and top_ids go together", who);
  if (top_ids) {
    k = top_ids->ndim == 2 ? top_ids->shape[1] : 0;
    if (k < 1 || k > V) return fail(MABA_ERR_INVALID, "%s: between 1 and V alternatives, in [%lld, k]", who, (long long)R);
    if (k > 64) return fail(MABA_ERR_UNSUPPORTED, "%s: at most 64 alternatives", who);
    for (const maba_tensor* t : {(const maba_tensor*)top_logp, (const maba_tensor*)top_ids}) {
      if (t->dtype != (t == top_ids ? MABA_I64 : MABA_F32)) return fail(MABA_ERR_DTYPE, "%s: top_logp is f32 and top_ids i64", who);
      if (t->ndim != 2 || t->shape[0] != R || t->shape[1] != k || (R > 1 && t->stride[0] != k) || (k > 1 && t->stride[1] != 1) ||
          (R > 0 && !t->data))
        return fail(MABA_ERR_INVALID, "%s: top_logp and top_ids must be contiguous [%lld, %lld]", who, (long long)R, (long long)k);
    }
  }
  if (R == 0) return MABA_OK;
  const ForwardArgs a = {logits_of(logits), (const int64_t*)targets->data, (float*)logp->data, (float*)entropy->data, (float*)lse->data,
                         k ? (float*)top_logp->data : nullptr, k ? (int64_t*)top_ids->data : nullptr, R, (int)V, (int)k,
                         (float)(1.0 / temperature)};
  const bool small = V <= 4096;
  const dim3 grid((unsigned)(small ? ceil_div(R, 4) : R)), block(small ? 256 : 512);
  auto run = [&](auto type) {
    typedef decltype(type) T;
    auto kernel = small ? (k ? logprobs_kernel<T, 1, true> : logprobs_kernel<T, 1, false>)
                        : (k ? logprobs_kernel<T, 8, true> : logprobs_kernel<T, 8, false>);
    hipLaunchKernelGGL(kernel, grid, block, 0, (hipStream_t)stream, a);
  };
  if (logits->dtype == MABA_F32) run(F32());
  else if (logits->dtype == MABA_BF16) run(Bf16());
  else run(Fp16());
  return check_launch(who);
}

extern "C" int maba_hip_token_logprobs_backward(const maba_tensor* dlogp, const maba_tensor* dentropy, const maba_tensor* dlse,
                                                const maba_tensor* logits, const maba_tensor* targets, const maba_tensor* lse,
                                                const maba_tensor* entropy, double temperature, maba_tensor* dlogits, void* stream) {
  const char* who = "token_logprobs_backward";
  int64_t R = 0, R2 = 0;
  int rc = check_logits(logits, who, "logits", R);
  if (!rc) rc = check_logits(dlogits, who, "dlogits", R2);
  if (!rc && !(temperature > 0.0 && 1.0 / temperature <= 1e30 && 1.0 / temperature >= 1e-30))
    rc = fail(MABA_ERR_INVALID, "%s: temperature=%g must be positive", who, temperature);
  if (!rc) rc = check_row_vec(targets, who, "targets", MABA_I64, R);
  if (!rc) rc = check_row_vec(lse, who, "lse", MABA_F32, R);
  if (!rc) rc = check_row_vec(entropy, who, "entropy", MABA_F32, R);
  if (!rc && dlogp) rc = check_row_vec(dlogp, who, "dlogp", MABA_F32, R);
  if (!rc && dentropy) rc = check_row_vec(dentropy, who, "dentropy", MABA_F32, R);
  if (!rc && dlse) rc = check_row_vec(dlse, who, "dlse", MABA_F32, R);
  if (rc) return rc;
  const int64_t V = logits->shape[logits->ndim - 1];
  if (dlogits->dtype != logits->dtype) return fail(MABA_ERR_DTYPE, "%s: dlogits must have the logits' type", who);
  if (R2 != R || dlogits->shape[dlogits->ndim - 1] != V) return fail(MABA_ERR_INVALID, "%s: dlogits must have the logits' rows", who);
  for (int i = 0; i + 1 < dlogits->ndim; ++i)
    if (dlogits->shape[i] > 1 && dlogits->stride[i] < (i + 2 == dlogits->ndim ? V : dlogits->shape[1] * dlogits->stride[1]))
      return fail(MABA_ERR_INVALID, "%s: rows of dlogits overlap", who);
  if (R > 0 && overlap(logits, dlogits)) {
    bool same = logits->data == dlogits->data && logits->ndim == dlogits->ndim;
    for (int i = 0; same && i + 1 < logits->ndim; ++i)
      same = logits->shape[i] == dlogits->shape[i] && (logits->shape[i] <= 1 || logits->stride[i] == dlogits->stride[i]);
    if (!same) return fail(MABA_ERR_INVALID, "%s: logits and dlogits overlap", who);
  }
  if (R == 0) return MABA_OK;
  const int64_t chunks = ceil_div(V, logits->dtype == MABA_F32 ? 4 : 8);
  BackwardArgs a = {logits_of(logits), logits_of(dlogits), (const int64_t*)targets->data,
                    dlogp ? (const float*)dlogp->data : nullptr, dentropy ? (const float*)dentropy->data : nullptr,
                    dlse ? (const float*)dlse->data : nullptr, (const float*)lse->data, (const float*)entropy->data, R, (int)V, 6, 1,
                    (float)(1.0 / temperature)};
  while (a.lg < 8 && chunks > (int64_t)4 << a.lg) ++a.lg;
  a.parts = (int)std::min<int64_t>(ceil_div(chunks, 256 * 8), 0x7fffffff / R);
  const dim3 grid((unsigned)(ceil_div(R, 256 >> a.lg) * a.parts));
  auto kernel = logits->dtype == MABA_F32 ? logprobs_back_kernel<F32> : logits->dtype == MABA_BF16 ? logprobs_back_kernel<Bf16>
                                                                                                  : logprobs_back_kernel<Fp16>;
  hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, a);
  return check_launch(who);
}
