// Log probabilities of given tokens, the entropy of their distributions and the likeliest alternatives, from logits
// [rows, V], and the gradient of the first two and of the normaliser.  With u = l / T:
//   lse = log sum exp(u),  logp = u[t] - lse,  H = lse - sum p u,  p = exp(u - lse)
//   dl  = 1/T (dlogp (delta_t - p) + dlse p - dH p (log p + H)),  and for the target 1 - p = the sum of the others' p
//
// Forward is one pass with a running reference: a thread holds (R, S, D) = (R, sum 2^x, sum x 2^x), x = l c - R, c = log2(e) / T,
// with R the largest l c so far rounded up to a whole number, so that l c - R is one fused operation without a rounding of R
// of its own, and two such triples over different elements join by a shift.  Then lse = ln 2 (R + log2 S), logp =
// ln 2 (l c - R - log2 S) and H = ln 2 (log2 S - D / S): differences from the reference, so that nothing large cancels.
//
// Alternatives: the k-th largest, or so, of the threads' own largest elements is a bound with no fewer than k elements at or
// above it.  The threads that have any collect theirs, some tens in all, and one wave sorts them.  The order is by
// value and then the lower index, so ties have one answer.
//
// Bound: HBM; forward reads the logits once, backward reads them and writes their gradient.
#include "row_vec.h"
#include "topk_wave.h"

namespace maba {
namespace logprobs {

using namespace rowvec;

constexpr float LOWEST = -3.40282347e38f, LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

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
  int64_t first, R;                  // rows first to R - 1
  int V, k;
  float inv;                         // 1 / T
};

// The order of alternatives: by value (NaN above all, -0 as +0), then the lower index.
__device__ __forceinline__ key64 order_key(float v, uint32_t idx) {
  const uint32_t o = v != v ? 0xffffffffu : order_f32(v + 0.f);
  return ((key64)o << 32) | (key64)(~idx);
}

// R is a whole number of at least FLOOR.  Up to -FLOOR the product that it is rounded up from is off by 64 at most, and 2^x
// stays in range; elements far below FLOOR have no part in S.
constexpr float FLOOR = -1073741824.f;
struct Triple { float r, s, d; };
// (s, d) with the reference raised by -by, f = 2^by.  by may be past fp32's range, and f is zero then.
__device__ __forceinline__ void raise(float& s, float& d, float by) {
  const float f = __builtin_amdgcn_exp2f(by);
  d = fmaf(d, f, fmaxf(by, LOWEST) * f * s);
  s *= f;
}
__device__ __forceinline__ Triple join(Triple a, Triple b) {
  const float r = fmaxf(a.r, b.r);
  raise(a.s, a.d, a.r - r);
  raise(b.s, b.d, b.r - r);
  return {r, a.s + b.s, a.d + b.d};
}

// Of all lanes of a wave.
__device__ __forceinline__ Triple wave_join(Triple t) {
  t = join(t, {peer<0>(t.r), peer<0>(t.s), peer<0>(t.d)});
  t = join(t, {peer<1>(t.r), peer<1>(t.s), peer<1>(t.d)});
  t = join(t, {peer<2>(t.r), peer<2>(t.s), peer<2>(t.d)});
  t = join(t, {peer<3>(t.r), peer<3>(t.s), peer<3>(t.d)});
  Pair r = both<false>(t.r), s = both<false>(t.s), d = both<false>(t.d);
  t = join({r.a, s.a, d.a}, {r.b, s.b, d.b});
  r = both<true>(t.r), s = both<true>(t.s), d = both<true>(t.d);
  return join({r.a, s.a, d.a}, {r.b, s.b, d.b});
}
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }

// The running state of a thread over its elements, and the largest of them; with TOP also where the round of elements is that
// has it, and the largest of the other rounds.
template <bool TOP>
struct Running {
  Triple t = {FLOOR, 0.f, 0.f};
  float best = -INFINITY, other = -INFINITY;
  int where = 0;
  template <int N>
  __device__ __forceinline__ void take(const float (&v)[N], int first, float c) {
    float b = TOP ? -INFINITY : best;
#pragma unroll
    for (int e = 0; e < N; ++e) b = fmaxf(b, v[e]);
    if constexpr (TOP) {
      other = fmaxf(other, fminf(best, b));
      where = b > best ? first : where;
      b = fmaxf(best, b);
    }
    best = b;
    const float r = fmaxf(t.r, ceilf(b * c));
    raise(t.s, t.d, t.r - r);
    t.r = r;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float x = fmaf(v[e], c, -r), p = __builtin_amdgcn_exp2f(x);
      t.s += p;
      t.d = fmaf(fmaxf(x, LOWEST), p, t.d);          // -inf times a p of zero is zero here
    }
  }
};

// The n-th largest (from 1) of a wave's values.
__device__ __forceinline__ float nth_of_wave(float v, int n) {
  const int lane = threadIdx.x & 63;
  if (n <= 8) {                                        // take the largest out n times; beyond that sorting is shorter
    float m = v;
    for (int i = 0;; ++i) {
      m = wave_joined(v, larger);
      if (i == n - 1) return m;
      const uint64_t at = __ballot(v == m);
      if (lane == __builtin_ctzll(at)) v = -INFINITY;
    }
  }
#pragma unroll
  for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor(v, j);
      v = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(v, o) : fminf(v, o);
    }
  return __shfl(v, n - 1);
}

template <class T>
__device__ __forceinline__ float element(const char* row, uint32_t i) {
  float w[Traits<T>::VEC];
  unpack<T>(load_chunk<T>(row, i * (16 / Traits<T>::VEC), 1), w);
  return w[0];
}

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

// v of all W waves' lanes joined.
template <int W, class F>
__device__ __forceinline__ float across(float v, float* shared, F f) {
  v = wave_joined(v, f);
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    v = shared[0];
#pragma unroll
    for (int w = 1; w < W; ++w) v = f(v, shared[w]);
  }
  return v;
}

// W waves a row (row_waves says how many).  With one, a workgroup has four rows; otherwise it is one row's.
// By itself and without alternatives 8,192 x 32,768 bf16 take 98 us, 5.5 TB/s: HBM; 777 x 50,257 fp32, whose rows start at any 4
// bytes, 34 us, 4.7 TB/s, and with eight alternatives 37.  (Behind a kernel that has just written as much, as a training step's
// gradient, the cache in front of HBM writes back meanwhile: 130 and, with the alternatives, 53.)  With them the threads that hold one
// read elements again, and the other waves of the row wait: 4,096 x 32,768 bf16 51 us without, 60 with 5 and 65 with 20 (4.5 and
// 4.2 TB/s; 65 and 71 where a thread read all of its elements again, a line of 128 bytes for 16).  16 x 32,768 take 5.3 and with 20
// alternatives 9.4 us, the latency of one row; 17 where all but five logits are -inf.
// CAP: room for what is above the bound.  Two lists of 1,024 a row of two waves held the compute unit to ten rows: 4,096 x
// 16,000 with five alternatives 46 us, with 512 43.
template <class T, int W, bool TOP>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void logprobs_kernel(ForwardArgs a) {
  constexpr int E = Traits<T>::VEC, NB = 32 / E, LANES = 64 * W, GROUPS = W == 1 ? 4 : 1, CAP = W > 4 ? 1024 : 256 * W;
  __shared__ Triple s_t[W];
  __shared__ float s_nth[W];
  __shared__ key64 s_above[TOP ? GROUPS * CAP : 1], s_equal[TOP ? GROUPS * CAP : 1];
  __shared__ int s_count[GROUPS][2];
  __shared__ float s_far[3][W];
  const int group = W == 1 ? threadIdx.x >> 6 : 0, lane = threadIdx.x & (LANES - 1), wave = W == 1 ? 0 : threadIdx.x >> 6;
  const int64_t r = a.first + (int64_t)blockIdx.x * GROUPS + __builtin_amdgcn_readfirstlane(group);
  if (W == 1 && r >= a.R) return;               // nothing below waits for another wave where W is 1
  const char* row = a.x.row(r);
  const float c = a.inv * LOG2E;
  const int64_t target = a.targets[r];
  float lt = 0.f;
  if (target >= 0 && target < a.V) lt = element<T>(row, (uint32_t)target);
  Running<TOP> run;
  for_chunks<T, NB>(row, a.V, lane, LANES, [&](auto& v, int first) { run.take(v, first, c); });
  Triple t = wave_join(run.t);
  float bound = 0.f;
  if constexpr (TOP) {
    // each of W waves has k / W elements at or above its own k / W-th largest, and so all have k at or above the least of those
    bound = nth_of_wave(run.best, (a.k + W - 1) / W);
    if (lane < 2) s_count[group][lane] = 0;
  }
  if constexpr (W > 1) {
    if ((threadIdx.x & 63) == 0) {
      s_t[wave] = t;
      s_nth[wave] = bound;
    }
    __syncthreads();
    t = s_t[0];
    bound = s_nth[0];
#pragma unroll
    for (int w = 1; w < W; ++w) {
      t = join(t, s_t[w]);
      bound = fminf(bound, s_nth[w]);
    }
  }
  // No sum, or none that is a number, or a reference out of range: every logit is -inf, or one is NaN or +inf, or the
  // largest is far from zero, as where a mask of the type's lowest value leaves nothing else.  Again, then, from the largest itself.
  const bool far = !(t.s > 0.f) || t.r > -FLOOR;
  float m = 0.f;
  if (far) {
    m = -INFINITY;
    for_chunks<T, 1>(row, a.V, lane, LANES, [&](auto& v, int) {
#pragma unroll
      for (int e = 0; e < E; ++e) m = fmaxf(m, v[e]);
    });
    m = across<W>(m, s_far[0], larger);
    m = m == -INFINITY ? 0.f : m;
    t = {0.f, 0.f, 0.f};
    for_chunks<T, 1>(row, a.V, lane, LANES, [&](auto& v, int) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float x = (v[e] - m) * c, p = __builtin_amdgcn_exp2f(x);
        t.s += p;
        t.d = fmaf(fmaxf(x, LOWEST), p, t.d);
      }
    });
    t.s = across<W>(t.s, s_far[1], sum_of);
    t.d = across<W>(t.d, s_far[2], sum_of);
  }
  const float log_s = __builtin_amdgcn_logf(t.s);
  const bool none = t.s == 0.f;                  // every logit is -inf: so are the log probabilities, and the entropy is 0
  float lse = far ? fmaf(m, a.inv, log_s * LN2) : (t.r + log_s) * LN2;
  if (!none) lse = lse < LOWEST ? LOWEST : lse > -LOWEST ? -LOWEST : lse;       // -inf says that there is no mass
  const auto logp_of = [&](float l) {
    const float v = ((far ? (l - m) * c : fmaf(l, c, -t.r)) - log_s) * LN2;
    // c is above 1 / T: a masked token's lowest value can leave fp32's range in base 2 alone
    return none ? -INFINITY : v == -INFINITY && l != -INFINITY ? fmaf(l, a.inv, -lse) : v;
  };
  if (lane == 0) {
    a.lse[r] = lse;
    a.entropy[r] = none ? 0.f : (log_s - t.d / t.s) * LN2;
    a.logp[r] = target < 0 ? 0.f : target >= a.V ? NAN : logp_of(lt);
  }
  if constexpr (TOP) {
    key64 *above = s_above + group * CAP, *equal = s_equal + group * CAP;
    int* count = s_count[group];
    // which of a chunk's elements are at or above the bound, or above it
    const auto at_least = [&](int at, bool strictly) {
      float v[E];
      unpack<T>(load_chunk<T>(row, (uint32_t)at * (16 / E), a.V - at), v);
      uint32_t hits = 0;
#pragma unroll
      for (int e = 0; e < E; ++e) hits |= v[e] < bound || (strictly && v[e] == bound) ? 0u : 1u << e;
      return hits;
    };
    // Most often one round of a thread's elements is enough.  (A thread whose sum is NaN may have NaN among its elements, which
    // its largest does not tell.)
    if (const bool all = run.other >= bound || run.t.s != run.t.s; all || run.best >= bound)
      for (int first = all ? lane * E : run.where, end = all ? a.V : first + 1; first < end; first += LANES * NB * E) {
        uint32_t hits = 0;
#pragma unroll
        for (int b = 0; b < NB; ++b) hits |= at_least(first + b * LANES * E, false) << (b * E);
        while (hits) {
          const int e = __builtin_ctz(hits), idx = first + (e / E) * LANES * E + e % E;
          hits &= hits - 1;
          if (idx >= a.V) continue;
          const float x = element<T>(row, (uint32_t)idx);
          const bool eq = x == bound;
          if (eq && *(volatile int*)&count[1] >= CAP) {        // more than will be read are not counted on
            uint32_t over = 0;
#pragma unroll 1
            for (int b = 0; b < NB; ++b) over |= at_least(first + b * LANES * E, true) << (b * E);
            hits &= over;
            continue;
          }
          const int at = atomicAdd(&count[eq], 1);
          if (at < CAP) (eq ? equal : above)[at] = order_key(x, (uint32_t)idx);
        }
      }
    if constexpr (W > 1) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int n = *(volatile int*)&count[0], ties = *(volatile int*)&count[1];
    const auto put = [&](int rank, key64 key) {
      a.top_ids[r * a.k + rank] = (int64_t)key_index(key);
      a.top_logp[r * a.k + rank] = logp_of(key_score(key));
    };
    if (n <= CAP && (n >= a.k || ties < CAP)) {
      // an element's place is the number of those ahead of it; equal ones come behind those above the bound
      for (int j = lane; j < n; j += LANES) {
        const key64 key = above[j];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += above[i] > key;
        if (rank < a.k) put(rank, key);
      }
      if (n < a.k)
        for (int j = lane; j < ties; j += LANES) {
          const key64 key = equal[j];
          int rank = n;
          for (int i = 0; i < ties; ++i) rank += equal[i] > key;
          if (rank < a.k) put(rank, key);
        }
      return;
    }
    const int l = threadIdx.x & 63;
    key64 list = KEY_NONE;
    if (n <= CAP) {
      if (wave != 0) return;
      // many of one value: the first ones of the row, in order
      for (int i = 0; i < n; i += 64) list = wave_merge_topk(list, i + l < n ? above[i + l] : KEY_NONE, 64);
      for (int i = 0, found = n; i < a.V && found < a.k; i += 64) {
        const float v = i + l < a.V ? element<T>(row, (uint32_t)(i + l)) : NAN;
        found += __popcll(__ballot(v == bound));
        list = wave_merge_topk(list, v == bound ? order_key(v, (uint32_t)(i + l)) : KEY_NONE, 64);
      }
    } else {
      // more above the bound than there is room for: a row whose largest elements are a few threads' own.  Each wave sorts
      // its part, an element of each lane at a time (16 rows of 32,768 rising logits, k = 20: 41 us; one wave alone 663)
      for (int c0 = 0; c0 * E < a.V; c0 += LANES) {
        const int first = (c0 + lane) * E, left = a.V - first;
        float v[E];
        unpack<T>(load_chunk<T>(row, (uint32_t)(c0 + lane) * 16u, left), v);
        uint32_t hits = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) hits |= e >= left || v[e] < bound ? 0u : 1u << e;
        while (__any(hits != 0)) {
          const uint32_t idx = (uint32_t)(first + __builtin_ctz(hits | 0x80000000u));
          list = wave_merge_topk(list, hits ? order_key(element<T>(row, idx), idx) : KEY_NONE, a.k);
          hits &= hits - 1;
        }
      }
      if constexpr (W > 1) {
        above[threadIdx.x] = list;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll 1
        for (int w = 1; w < W; ++w) list = wave_merge_topk(list, above[64 * w + l], a.k);
      }
    }
    if (l < a.k) put(l, list);
  }
}

struct BackwardArgs {
  Logits x, dx;
  const int64_t* targets;
  const float *dlogp, *dentropy, *dlse, *lse, *entropy;
  int64_t first, R;                  // rows first to R - 1
  int V, lg, parts;                  // 2^lg threads a row, 64 or 256, and `parts` workgroups side by side on it
  float inv;
};

// One read and one write of the logits: 8,192 x 32,768 bf16 194 us, 777 x 50,257 fp32 57 us, both 5.5 TB/s: HBM.  Long rows go
// to several workgroups, eight chunks a thread, so that few of them fill the chip too: 16 x 32,768 5.6 us.
template <class T>
__global__ __launch_bounds__(256) void logprobs_back_kernel(BackwardArgs a) {
  constexpr int E = Traits<T>::VEC, NB = 2;
  const int64_t r = a.first + (int64_t)blockIdx.x / a.parts * (256 >> a.lg) + __builtin_amdgcn_readfirstlane(threadIdx.x >> a.lg);
  if (r >= a.R) return;
  const char* row = a.x.row(r);
  char* out = (char*)a.dx.row(r);
  const int64_t target = a.targets[r];
  float lse = a.lse[r];
  const float h = a.entropy[r];
  float gh = a.dentropy ? a.dentropy[r] : 0.f;
  float gl = target < 0 || !a.dlogp ? 0.f : target >= a.V ? NAN : a.dlogp[r], gz = a.dlse ? a.dlse[r] : 0.f;
  // log p = l / T - lse is as exact as lse, whose rounding far from zero is more than those of p and of the result: there the
  // row is summed again and log p counted from its largest element.  All of that ends before anything of the row is
  // written, which may be the logits' own.  Each of a row's workgroups does so for itself.  (1,024 x 32,768 bf16, two of them, 23 us
  // without such rows and 61 with nothing else; 777 x 50,257 fp32, seven, 53 and 359.)
  constexpr float EXACT = T::CODE == MABA_F32 ? 32.f : 256.f;
  __shared__ float part[3][4];
  const int l = threadIdx.x & ((1 << a.lg) - 1);
  const auto of_row = [&](float v, float* shared, auto f) { return a.lg == 8 ? across<4>(v, shared, f) : wave_joined(v, f); };
  float m = 0.f;
  if (lse == -INFINITY) {            // no mass: no element has a gradient
    lse = -LOWEST;
    gl = gh = gz = 0.f;              // whatever comes from a loss of lse = -inf
  } else if (fabsf(lse) > EXACT) {
    m = -INFINITY;
    for_chunks<T, 2>(row, a.V, l, 1 << a.lg, [&](auto& v, int) {
#pragma unroll
      for (float x : v) m = fmaxf(m, x);
    });
    m = of_row(m, part[0], larger);
    float s = 0.f;
    for_chunks<T, 2>(row, a.V, l, 1 << a.lg, [&](auto& v, int) {
#pragma unroll
      for (float x : v) s += __builtin_amdgcn_exp2f((x - m) * a.inv * LOG2E);
    });
    lse = __builtin_amdgcn_logf(of_row(s, part[1], sum_of)) * LN2;
  }
  const int lanes = a.parts << a.lg, lane = ((int)(blockIdx.x % a.parts) << a.lg) + l;
  const int mine = target >= 0 && target < a.V ? (int)(target / E) : -1, chunks = (a.V + E - 1) / E;
  // The target's element has dlogp (1 - p) and dH p (log p + H).  Of a likely target 1 - p and log p are little more than lse's
  // rounding: below `sure`, where that is more than an eighth of a 16-bit result's half step (32 of an fp32 one's), 1 - p is
  // the sum of the others' p instead, made by the workgroup that has the element, before the row is written.  Only a row of
  // little entropy can hold such a target.  (8,192 x 32,768 bf16 194 us without such targets, 231 with nothing else.)
  constexpr float SHARE = T::CODE == MABA_F32 ? 32.f : T::CODE == MABA_BF16 ? 2048.f : 256.f;
  const float sure = fminf((fabsf(lse) + 4.f) / SHARE, 0.5f);
  float rest = -1.f;
  if (mine >= 0 && (gl != 0.f || gh != 0.f) && h < sure * (2.f + __logf((float)a.V / sure))) {
    const float at = element<T>(row, (uint32_t)target);
    if (a.lg == 8) __syncthreads();  // all waves have it before one of them writes the row
    if (-expm1f(fmaf(at - m, a.inv, -lse)) < sure && mine % lanes >> a.lg == (int)(blockIdx.x % a.parts)) {
      float s = 0.f;
      for_chunks<T, 2>(row, a.V, l, 1 << a.lg, [&](auto& v, int first) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(v) / sizeof(float)); ++i) {
          const float p = __builtin_amdgcn_exp2f(fmaf(v[i] - m, a.inv, -lse) * LOG2E);
          s += first + (i / E << a.lg) * E + i % E == (int)target ? 0.f : p;
        }
      });
      rest = of_row(s, part[2], sum_of);
    }
  }
  const float base = gz - gl - (gh != 0.f ? gh * h : 0.f), at_target = gl * a.inv;
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
        const float lp = fmaf(v[e] - m, a.inv, -lse), p = __builtin_amdgcn_exp2f(lp * LOG2E);
        // where p is zero log p may be -inf: bounded, its product with p is zero
        v[e] = a.inv * p * fmaf(-gh, fmaxf(lp, -1e4f), base);
      }
      if (ch == mine) {
        const float own = a.inv * fmaf(gl, rest, (1.f - rest) * (gz - (gh != 0.f ? gh * (log1pf(-rest) + h) : 0.f)));
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = e != (int)(target % E) ? v[e] : rest < 0.f ? v[e] + at_target : own;
      }
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
  for (int i = 0; i + 1 < n; ++i) {
    if (t->shape[i] < 0) return fail(MABA_ERR_INVALID, "%s: %s has a negative size", who, name);
    if (t->shape[i] > 0x7fffffff) return fail(MABA_ERR_UNSUPPORTED, "%s: too many rows", who);
  }
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
// Waves a row, of 1, 2, 4 and 8.  Many rows: as few as leave a thread 16 chunks, since what a row costs besides its elements
// (its waves' sums joined, the barriers) grows with them.  Few rows: as many as leave each thread a chunk, while all
// rows' waves are at most eight a compute unit.  In us for bf16 with five alternatives, 1 / 2 / 4 / 8 waves:
//   4,096 x 8,000   23 / 24 / 29 / 46    4,096 x 32,768   75 / 64 / 60 / 67    4,096 x 65,536   145 / 119 / 112 / 106
//   16 x 2,000      7.4 / 5.7 / 5.9 / 27 (waves without a chunk bound nothing)     16 x 32,768      20 / 12 / 9.7 / 8.3
static int row_waves(int64_t rows, int64_t chunks) {
  int w = 1;
  while (w < 8 && chunks > 16 * 64 * w) w *= 2;
  while (w < 8 && chunks >= 2 * 64 * w && rows * 2 * w <= 8 * (int64_t)device_cu_count()) w *= 2;
  return w;
}
// f(first row, one past the last) over the rows in launches of less than 2^32 threads, of which 64 to 512 work on a row.
constexpr int64_t MOST_ROWS = (int64_t)1 << 22;
template <class F>
static void in_launches(int64_t R, F f) {
  for (int64_t r = 0; r < R; r += MOST_ROWS) f(r, std::min(R, r + MOST_ROWS));
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
  ForwardArgs a = {logits_of(logits), (const int64_t*)targets->data, (float*)logp->data, (float*)entropy->data, (float*)lse->data,
                         k ? (float*)top_logp->data : nullptr, k ? (int64_t*)top_ids->data : nullptr, 0, R, (int)V, (int)k,
                         (float)(1.0 / temperature)};
  const int waves = row_waves(R, ceil_div(V, logits->dtype == MABA_F32 ? 4 : 8));
  const dim3 block(waves == 1 ? 256 : 64 * waves);
  auto run = [&](auto type) {
    typedef decltype(type) T;
    auto go = [&](auto kernel) {
      in_launches(R, [&](int64_t first, int64_t end) {
        a.first = first;
        a.R = end;
        const int64_t rows = end - first;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(waves == 1 ? ceil_div(rows, 4) : rows)), block, 0, (hipStream_t)stream, a);
      });
    };
    if (waves == 1) go(k ? logprobs_kernel<T, 1, true> : logprobs_kernel<T, 1, false>);
    else if (waves == 2) go(k ? logprobs_kernel<T, 2, true> : logprobs_kernel<T, 2, false>);
    else if (waves == 4) go(k ? logprobs_kernel<T, 4, true> : logprobs_kernel<T, 4, false>);
    else go(k ? logprobs_kernel<T, 8, true> : logprobs_kernel<T, 8, false>);
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
                    dlse ? (const float*)dlse->data : nullptr, (const float*)lse->data, (const float*)entropy->data, 0, R, (int)V, 6, 1,
                    (float)(1.0 / temperature)};
  // four waves a row, or one (us, one / four: 8,192 x 2,100 bf16 17.9 / 23.3, x 4,000 24.4 / 24.1, 300 x 4,000 6.4 / 5.0)
  if (chunks > (R > 4 * (int64_t)device_cu_count() ? 512 : 256)) a.lg = 8;
  a.parts = (int)std::min<int64_t>(ceil_div(chunks, 256 * 8), std::max<int64_t>(MOST_ROWS / R, 1));
  if (logits->data == dlogits->data) a.parts = 1;
  auto kernel = logits->dtype == MABA_F32 ? logprobs_back_kernel<F32> : logits->dtype == MABA_BF16 ? logprobs_back_kernel<Bf16>
                                                                                                  : logprobs_back_kernel<Fp16>;
  in_launches(R, [&](int64_t first, int64_t end) {
    a.first = first;
    a.R = end;
    hipLaunchKernelGGL(kernel, dim3((unsigned)(ceil_div(end - first, 256 >> a.lg) * a.parts)), dim3(256), 0, (hipStream_t)stream, a);
  });
  return check_launch(who);
}
