// Log-probabilities of tokens through the output head and the clipped policy loss on them: the
// logits products (tcgen05 GEMM core) with their epilogues, and the row kernels between them.
//
//   logp_t = logit_t[y_t] - lse_t                      d logp_t / d logit_t = onehot(y_t) - softmax
//   r_t = exp(logp_t - old_t)
//   loss = sum_t w_t ( -min(r_t A_t, clip(r_t, 1 - lo, 1 + hi) A_t) + kl_coef (e^d - d - 1) ),  d = ref_t - logp_t
//   w_t = 1 / tokens, or 1 / (sequences * tokens of t's sequence)
#include <type_traits>

#include "gemm_sm100.cuh"

namespace bt {
namespace {

constexpr int kThreads = 256;

bool rows_aligned(const void* p, int64_t ld, int elem_bytes) {
  return p != nullptr && aligned16(p) && (ld * elem_bytes) % 16 == 0;
}
bool aligned8(const void* p) { return reinterpret_cast<uintptr_t>(p) % 8 == 0; }  // statistics are pairs of floats
bool known(int dtype) { return dtype == BT_BF16 || dtype == BT_FP16 || dtype == BT_FP32; }
int esize(int dtype) { return dtype == BT_FP32 ? 4 : 2; }
__device__ __forceinline__ bool counted(int64_t label, int64_t ignore_index, int64_t vocab) {
  return label != ignore_index && label >= 0 && label < vocab;
}

// (max, sum exp) of a row from its half tiles; all lanes of the warp get the result.  Two passes, eight
// loads of a lane in flight: a running (max, sum) waits for each load and exponential in turn (1187 half
// tiles: 8.0 -> 5.0 us for 61 rows).
__device__ __forceinline__ float2 merge_stats(const float2* __restrict__ ts, int n_vt, int lane) {
  constexpr int kAhead = 8;
  float mx = -1e30f, sum = 0.f;
  for (int i0 = lane; i0 < n_vt; i0 += 32 * kAhead) {
    float x[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) x[u] = i0 + u * 32 < n_vt ? ts[i0 + u * 32].x : -1e30f;
#pragma unroll
    for (int u = 0; u < kAhead; ++u) mx = fmaxf(mx, x[u]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  for (int i0 = lane; i0 < n_vt; i0 += 32 * kAhead) {
    float2 t[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) t[u] = i0 + u * 32 < n_vt ? ts[i0 + u * 32] : make_float2(-1e30f, 0.f);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) sum += t[u].y * __expf(t[u].x - mx);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  return make_float2(mx, sum);
}

// target - lse.  (target - max) is exact near the maximum, where a rounding of max + log(sum) would
// show; both callers take this, so that the ratio of a policy to itself is exactly 1.
__device__ __forceinline__ double log_prob(float target, float2 st) {
  return static_cast<double>(target - st.x) - log(static_cast<double>(st.y));
}

// One warp per row: lse and log-probability (0 where the position does not count).
__global__ void __launch_bounds__(kThreads)
logp_rows_kernel(const float2* __restrict__ tile_stats, const float* __restrict__ tgt_logit,
                 const int64_t* __restrict__ labels, float* __restrict__ logp, float* __restrict__ lse, int64_t rows,
                 int n_vt, int64_t ignore_index, int64_t vocab, int32_t* __restrict__ status) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (static_cast<int64_t>(gridDim.x) * kThreads) >> 5;
  for (int64_t row = warp0; row < rows; row += nwarps) {
    const float2 st = merge_stats(tile_stats + row * n_vt, n_vt, lane);
    if (lane == 0) {
      const int64_t label = labels[row];
      const bool in = counted(label, ignore_index, vocab);
      if (!in && label != ignore_index && status != nullptr) atomicOr(status, BT_STATUS_BAD_LABEL);
      logp[row] = in ? static_cast<float>(log_prob(tgt_logit[row], st)) : 0.f;
      if (lse != nullptr) lse[row] = st.x + logf(st.y);
    }
  }
}

// fp16 holds dlogits = coef (onehot - softmax) between 2^-24 and 65504 only, while a coefficient may be
// anything: ratios and KL gaps are exponentials.  A row whose coefficient lies outside [1/2, 2^15) is
// therefore formed from coef 2^-e, which does not; the product with W gives that row's d hidden 2^e times
// in its fp32 epilogue, and the one with x takes the row of x times 2^(e - E), E not below any e so far,
// so that d weight comes out in units of 2^E.  What the row of x loses in fp16's subnormal steps, 2^-25
// 2^(E - e), is 2^-25 of what the largest rows contribute.  (All rows at [2^14, 2^15) would round the softmax at
// full precision down to 2^-28 instead of 2^-13, and cost 5% at 4096 and 16384 rows: digits cost power.)
__device__ __forceinline__ int row_exponent(double coef) {
  if (coef == 0.0 || !isfinite(coef)) return 0;
  int e;
  frexp(coef, &e);
  e = e > 15 ? e - 15 : min(e, 0);
  return max(-60, min(100, e));
}
// E goes up in steps of four, so that it seldom does from one chunk to the next.
__device__ __forceinline__ int step_of(int e) { return (e + 3) & ~3; }
constexpr int kNoExponent = -1000;  // E before the first coefficient

// Upstream gradient of the log-probabilities as the coefficients of the dlogits product, scaled by a
// power of two so that the largest is in [1/2, 1): with fp16 operands a mean over many tokens would
// otherwise push them, times the softmax, below the type's range.  scal[0] = scale back.  row_scale (fp16,
// else null): 2^e of each row, at most 1 here.
__global__ void __launch_bounds__(1024)
logp_coef_kernel(const float* __restrict__ dlogp, const int64_t* __restrict__ labels, int64_t n, int64_t ignore_index,
                 int64_t vocab, float* __restrict__ coef, float* __restrict__ row_scale, float* __restrict__ scal) {
  grid_dependency_wait();
  __shared__ float s_max[32];
  float mx = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024)
    if (counted(labels[i], ignore_index, vocab)) {
      const float a = fabsf(dlogp[i]);
      if (isfinite(a)) mx = fmaxf(mx, a);  // infinities and NaN keep their place, but set no scale
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = mx;
  __syncthreads();
  mx = s_max[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  int e = 0;
  if (mx > 0.f) frexpf(mx, &e);
  e = max(-125, min(125, e));
  const float up = ldexpf(1.f, -e);
  if (threadIdx.x == 0) scal[0] = ldexpf(1.f, e);
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    float c = counted(labels[i], ignore_index, vocab) ? dlogp[i] * up : 0.f;
    if (row_scale != nullptr) {
      const int e = row_exponent(c);
      c = ldexpf(c, -e);
      row_scale[i] = ldexpf(1.f, e);
    }
    coef[i] = c;
  }
}

// Rows of `x` that count, copied; zeros in the place of the others, which meet zero coefficients in
// the weight gradient's product and must be finite there.  For the policy loss (`scal` of
// policy_weights_kernel) rows behind the last sequence do not count, and with bad offsets none does.  For the
// log-probabilities (`row_scale`, or null) rows are multiplied by 2^e: E is 0, all coefficients being known.
template <typename T>
__global__ void __launch_bounds__(kThreads)
logp_mask_rows_kernel(const T* __restrict__ x, T* __restrict__ y, const int64_t* __restrict__ labels, int64_t rows,
                      int64_t h, int64_t ld, int64_t ignore_index, int64_t vocab, const float* __restrict__ scal,
                      const int32_t* __restrict__ cu, int n_seq, const float* __restrict__ row_scale) {
  grid_dependency_wait();
  constexpr int E = Cvt<T>::N;
  const int64_t nvec = h / E;
  int64_t covered = rows;
  if (scal != nullptr) covered = scal[1] == 0.f ? 0 : (cu != nullptr ? cu[n_seq] : rows);
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const bool in = row < covered && counted(labels[row], ignore_index, vocab);
    const float f = in && row_scale != nullptr ? row_scale[row] : 1.f;
    for (int64_t i = threadIdx.x; i < nvec; i += kThreads) {
      uint4 u = in ? ld_stream_v4(x + row * ld + i * E) : make_uint4(0, 0, 0, 0);
      if (f != 1.f) {
        float v[E];
        Cvt<T>::unpack(u, v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= f;
        u = Cvt<T>::pack(v);
      }
      st_global_v4(y + row * h + i * E, u);
    }
  }
}

// ------------------------------------------------------------------ the policy loss
// Weight of a counted token of each sequence (one entry for all tokens without offsets), and
// scal[0] = largest weight, scal[1] = 1 / that: coefficients are stored relative to it.  Where nothing
// counts (bad offsets among the reasons) scal[1] is 0.
__global__ void __launch_bounds__(1024)
policy_weights_kernel(const int64_t* __restrict__ labels, int64_t n, const int32_t* __restrict__ cu, int n_seq,
                      int64_t ignore_index, int64_t vocab, float* __restrict__ weights, float* __restrict__ scal,
                      int32_t* __restrict__ top_exp, int32_t* __restrict__ status) {
  grid_dependency_wait();
  __shared__ int s_filled, s_least;
  const int tid = threadIdx.x, lane = tid & 31;
  if (tid == 0) s_filled = 0, s_least = 0x7fffffff;
  bool bad_label = false, bad_cu = false;
  for (int64_t i = tid; i < n; i += 1024) {
    const int64_t l = labels[i];
    bad_label |= l != ignore_index && (l < 0 || l >= vocab);
  }
  if (cu != nullptr)
    for (int i = tid; i < n_seq; i += 1024)
      bad_cu |= cu[i] < 0 || cu[i + 1] < cu[i] || cu[i + 1] > n || (i == 0 && cu[i] != 0);
  if (__syncthreads_or(bad_label) && tid == 0 && status != nullptr) atomicOr(status, BT_STATUS_BAD_LABEL);
  bad_cu = __syncthreads_or(bad_cu);
  if (bad_cu && tid == 0 && status != nullptr) atomicOr(status, BT_STATUS_BAD_SEQUENCES);
  for (int b = tid >> 5; b < n_seq; b += 32) {
    const int64_t lo = cu != nullptr ? cu[b] : 0, hi = cu != nullptr ? cu[b + 1] : n;
    int c = 0;
    if (!bad_cu)
      for (int64_t i = lo + lane; i < hi; i += 32) c += counted(labels[i], ignore_index, vocab) ? 1 : 0;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0) {
      weights[b] = __int_as_float(c);
      if (c > 0) {
        atomicAdd(&s_filled, 1);
        atomicMin(&s_least, c);
      }
    }
  }
  __syncthreads();
  for (int b = tid; b < n_seq; b += 1024) {
    const int c = __float_as_int(weights[b]);
    weights[b] = c > 0 ? static_cast<float>(1.0 / (static_cast<double>(c) * s_filled)) : 0.f;
  }
  if (tid == 0) {
    const double top = s_filled > 0 ? 1.0 / (static_cast<double>(s_least) * s_filled) : 1.0;
    scal[0] = static_cast<float>(top);
    scal[1] = s_filled > 0 ? static_cast<float>(1.0 / top) : 0.f;
    top_exp[0] = kNoExponent;
  }
}

struct PolicyArgs {
  const float2* tile_stats;
  const float* tgt_logit;
  const int64_t* labels;  // of this chunk
  const float* old_logp;
  const float* adv;
  const float* ref_logp;  // may be null
  const int32_t* cu;      // may be null
  const float* weights;
  const float* scal;
  float* logp;
  float* lse;
  float* coef;
  float* row_scale;  // fp16 gradients, else null: 2^e of each row (the memory of tgt_logit)
  int32_t* top_exp;  // E of this chunk, which starts as the one before
  float* terms;      // [3][total]: weighted loss, kl, clipped
  int64_t rows, row0, total, ignore_index, vocab;
  int n_vt, n_seq;
  float clip_low, clip_high, kl_coef;
};

// One warp per row.  The few operations on a row's scalars are done in fp64: e^d - d - 1 loses all its
// digits in fp32 when the policy is near its reference, and nothing here is bound by arithmetic.
__global__ void __launch_bounds__(kThreads)
policy_rows_kernel(const PolicyArgs a) {
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const int64_t warp0 = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5;
  const int64_t nwarps = (static_cast<int64_t>(gridDim.x) * kThreads) >> 5;
  for (int64_t row = warp0; row < a.rows; row += nwarps) {
    const float2 st = merge_stats(a.tile_stats + row * a.n_vt, a.n_vt, lane);
    if (lane != 0) continue;
    const int64_t g = a.row0 + row;
    float w = 0.f;
    if (counted(a.labels[row], a.ignore_index, a.vocab)) {
      int lo = 0;
      if (a.cu != nullptr) {  // the last sequence that starts at or before this token, if it reaches it
        int hi = a.n_seq;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (a.cu[mid] <= g) lo = mid;
          else hi = mid;
        }
        w = a.n_seq > 0 && g < a.cu[lo + 1] ? a.weights[lo] : 0.f;
      } else {
        w = a.weights[0];
      }
    }
    double logp = 0.0, term = 0.0, kl = 0.0, coef = 0.0;
    bool held = false;
    if (w != 0.f) {  // what the others hold - old log-probabilities, advantages - is never looked at
      logp = static_cast<float>(log_prob(a.tgt_logit[row], st));  // as it is reported and was stored as `old`
      const double adv = a.adv[g], r = exp(logp - static_cast<double>(a.old_logp[g]));
      const double lo_r = 1.0 - static_cast<double>(a.clip_low), hi_r = 1.0 + static_cast<double>(a.clip_high);
      held = (adv > 0.0 && r > hi_r) || (adv < 0.0 && r < lo_r);
      term = -adv * (held ? (adv > 0.0 ? hi_r : lo_r) : r);
      coef = held ? 0.0 : -adv * r;
      if (a.ref_logp != nullptr) {
        const double d = static_cast<double>(a.ref_logp[g]) - logp, em1 = expm1(d);
        kl = em1 - d;
        if (a.kl_coef != 0.f) {  // 0 is for the log alone: its infinity is not the loss's
          term += a.kl_coef * kl;
          coef -= a.kl_coef * em1;
        }
      }
    }
    a.logp[row] = static_cast<float>(logp);
    a.lse[row] = st.x + logf(st.y);
    coef = coef * w * static_cast<double>(a.scal[1]);
    if (a.row_scale != nullptr) {
      const int e = row_exponent(coef);
      if (coef != 0.0) atomicMax(a.top_exp, step_of(e));
      coef = ldexp(coef, -e);
      a.row_scale[row] = ldexpf(1.f, e);
    }
    a.coef[row] = static_cast<float>(coef);
    a.terms[g] = static_cast<float>(term * w);
    a.terms[a.total + g] = static_cast<float>(kl * w);
    a.terms[2 * a.total + g] = held ? w : 0.f;
  }
}

// loss, averages[0..1] = sums of the three rows of terms (fp64, fixed order); averages[4] = the scale of
// d weight, the largest token weight times 2^E.
__global__ void __launch_bounds__(1024)
policy_reduce_kernel(const float* __restrict__ terms, int64_t n, float* __restrict__ loss, float* __restrict__ averages,
                     const int32_t* __restrict__ top_exp) {
  grid_dependency_wait();
  __shared__ double s_sum[32];
  const float* t = terms + blockIdx.x * n;
  double a = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) a += static_cast<double>(t[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x == 0) {
    double s = 0.0;
    for (int i = 0; i < 32; ++i) s += s_sum[i];
    (blockIdx.x == 0 ? loss : averages + (blockIdx.x - 1))[0] = static_cast<float>(s);
    if (blockIdx.x == 0)
      averages[4] = top_exp != nullptr && *top_exp != kNoExponent ? ldexpf(averages[2], *top_exp) : averages[2];
  }
}

// Shifted logits -> coef (onehot - softmax), in place: one read and one write of the chunk, 16 bytes
// per thread and step.  exp(logit - lse) = exp(stored) exp(half-tile max - lse), the second factor
// once per vector.  Bound by memory: 1024 rows x 151936, 622 MB in 106 us, 5.9 TB/s; kept out of the products'
// epilogues because a row's lse needs all of its tiles.  fp16: also brings the rows of x to the common
// 2^E, and hands E to the next chunk.
struct Exponents {
  const float* row_scale;  // null: no fp16 gradients
  const int32_t* top;
  int32_t* next;
  void* x;
  int64_t h;
};
template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_dlogits_kernel(T* __restrict__ logits, const float2* __restrict__ tile_stats, const float* __restrict__ lse,
                      const int64_t* __restrict__ labels, const float* __restrict__ coef, int64_t rows, int64_t V,
                      int64_t ld, int n_vt, const Exponents ex) {
  grid_dependency_wait();
  constexpr int E = Cvt<T>::N;
  const int64_t nvec = (V + E - 1) / E;
  const int64_t seg = (nvec + gridDim.y - 1) / gridDim.y;
  const int64_t v_begin = static_cast<int64_t>(blockIdx.y) * seg;
  const int64_t v_end = v_begin + seg < nvec ? v_begin + seg : nvec;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const float c = coef[row], l = lse[row];
    const int64_t label = labels[row];
    const float2* ts = tile_stats + row * n_vt;
    T* lr = logits + row * ld;
    for (int64_t v = v_begin + threadIdx.x; v < v_end; v += kThreads) {
      const int64_t c0 = v * E;
      float f[E];
      if (c != 0.f) {
        const float scale = -c * __expf(ts[c0 >> 7].x - l);
        Cvt<T>::unpack(ld_stream_v4(lr + c0), f);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = __expf(f[e]) * scale;
        if (label >= c0 && label < c0 + E) {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (c0 + e == label) f[e] += c;
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = 0.f;
      }
      st_global_v4(lr + c0, Cvt<T>::pack(f));
    }
  }
  if constexpr (std::is_same<T, __half>::value) {
    if (ex.row_scale == nullptr || blockIdx.y != 0) return;
    const int top = *ex.top;
    if (blockIdx.x == 0 && threadIdx.x == 0) *ex.next = top;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
      const float f = coef[row] != 0.f ? ldexpf(ex.row_scale[row], -top) : 1.f;
      if (f == 1.f) continue;
      T* xr = static_cast<T*>(ex.x) + row * ex.h;
      for (int64_t i = threadIdx.x; i < ex.h / E; i += kThreads) {
        float v[E];
        Cvt<T>::unpack(ld_global_v4(xr + i * E), v);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] *= f;
        st_global_v4(xr + i * E, Cvt<T>::pack(v));
      }
    }
  }
}

// The sum of d weight over the chunks so far, brought to the units of the newest one; nothing to do while
// E has not grown.
__global__ void __launch_bounds__(kThreads)
policy_rescale_kernel(float* __restrict__ acc, int64_t n4, const int32_t* __restrict__ before,
                      const int32_t* __restrict__ now) {
  grid_dependency_wait();
  const int e0 = *before, e1 = *now;
  if (e0 == e1 || e0 == kNoExponent) return;  // (no coefficient so far: zeros)
  const float f = ldexpf(1.f, e0 - e1);
  float4* a = reinterpret_cast<float4*>(acc);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n4; i += step) {
    float4 v = a[i];
    v.x *= f, v.y *= f, v.z *= f, v.w *= f;
    a[i] = v;
  }
}

unsigned grid_for(int64_t blocks, int per_sm) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<unsigned>(blocks < 1 ? 1 : (blocks < cap ? blocks : cap));
}

// What the steps below share: one call's sizes, types and stream.
struct Head {
  const void* W;
  int64_t H, V, ld_logits, ignore_index;
  int dtype, n_vt;
  int32_t* status;
  cudaStream_t s;
};

// Whether the logits of `rows` rows are better computed in 128-row tiles, one CTA each, than in the
// 256-row tiles of CTA pairs: when the last pair tile is at least half empty and that half outweighs the
// pairs' advantage (their tiles read half as much of W each), 7 - 13% at whole numbers of pair tiles.
// Log-probabilities, forward, pairs / single CTAs, us: vocabulary 151936 x 4096, 61 rows 254 / 235, 128 rows
// 276 / 240, 129 rows 285 / 341, 384 rows 543 / 473, 512 rows 532 / 611, 640 rows 766 / 724, 1024 rows
// 1020 / 1093; 32000 x 1024, 640 rows 51 / 42.  (Tiles drawn at run time are the pairs' alone.)
bool narrow_tiles(int64_t rows) {
  return gemm::dynamic_tiles() == 0 &&
         ceil_div(rows, 128) * 128 * 1.1 < static_cast<double>(ceil_div(rows, 256) * 256);
}

gemm::Launch head_product(const Head& h, const void* hidden, const int64_t* labels, int64_t rows, int64_t ld_hidden) {
  gemm::Launch L;
  L.dtype = h.dtype;
  L.a0.ptr = hidden, L.a0.kmajor = 1, L.a0.mn = rows, L.a0.k = h.H, L.a0.ld = ld_hidden;
  L.b0.ptr = h.W, L.b0.kmajor = 1, L.b0.mn = h.V, L.b0.k = h.H, L.b0.ld = h.H;
  L.p.M = static_cast<int>(rows);
  L.p.N = static_cast<int>(h.V);
  L.p.status = h.status;
  L.p.labels = labels;
  L.p.ignore_index = h.ignore_index;
  L.p.n_vtiles = h.n_vt;
  L.single = narrow_tiles(rows);
  return L;
}

// Statistics (and, unless NULL, shifted logits) of one chunk.
int stats(const Head& h, const void* hidden, const int64_t* labels, void* logits, float* tile_stats, float* tgt,
          int64_t rows, int64_t ld_hidden) {
  gemm::Launch L = head_product(h, hidden, labels, rows, ld_hidden);
  L.p.tile_stats = tile_stats;
  L.p.tgt_logit = tgt;
  if (logits == nullptr) return gemm::launch<gemm::EPI_LOGP>(L, h.s);
  L.p.out = logits;
  L.p.ldo = h.ld_logits;
  L.p.vec_ok = rows_aligned(logits, h.ld_logits, esize(h.dtype));
  return gemm::launch<gemm::EPI_LOGP_SHIFT>(L, h.s);
}

int mask_rows(const Head& h, const void* x, void* y, const int64_t* labels, int64_t rows, int64_t ld,
              const float* scal, const int32_t* cu, int n_seq, const float* row_scale) {
  const dim3 grid(grid_for(rows, 8)), block(kThreads);
  const cudaError_t e =
      h.dtype == BT_FP32
          ? launch_dependent(logp_mask_rows_kernel<float>, grid, block, 0, h.s, static_cast<const float*>(x),
                             static_cast<float*>(y), labels, rows, h.H, ld, h.ignore_index, h.V, scal, cu, n_seq,
                             row_scale)
          // a copy, but for fp16's scales: the two 16-bit types are the same
          : launch_dependent(logp_mask_rows_kernel<__half>, grid, block, 0, h.s, static_cast<const __half*>(x),
                             static_cast<__half*>(y), labels, rows, h.H, ld, h.ignore_index, h.V, scal, cu, n_seq,
                             row_scale);
  BT_CHECK_LAUNCHED(e, "logp: copy of the counted rows");
  return BT_OK;
}

// Runs into which the contraction of d hidden is cut.  The result has few tiles (rows x H) against a long
// contraction (V): 517 x 1024 from V = 32000 is 12 tiles for 74 CTA pairs, 2048 x 4096 is 1.7 waves.
// The fewest runs that come within 3% of the least estimated time: waves of tiles at the sustained
// product rate, and 8 bytes an element and run for the partial sums.  Measured, both gradient products
// together: 517 x 1024 x 32000 in 1 / 2 / 4 / 6 / 8 runs 201 / 126 / 90 / 78 / 94 us (6 taken);
// 4096 x 4096 x 151936 in 1 / 2 / 4 runs 8.05 / 7.59 / 7.69 ms (2 taken).
int dhidden_runs(int64_t rows, int64_t H, int64_t V, int dtype) {
  const int64_t pairs = sm_count() / 2, tiles = ceil_div(rows, 256) * ceil_div(H, 256);
  const int64_t blocks = ceil_div(V, 128 / esize(dtype));
  const double tile_s = 2.0 * 256 * 256 * V / (1.4e15 / 74);
  double least = 0.0, cost[17] = {};
  for (int s = 1; s <= 16; ++s) {
    const int64_t per = ceil_div(blocks, s);
    if (s > 1 && (per < 16 || ceil_div(blocks, per) != s)) continue;
    cost[s] = static_cast<double>(ceil_div(tiles * s, pairs)) * tile_s * per / blocks +
              (s > 1 ? s * rows * H * 8.0 / 6.5e12 + 2e-6 : 0.0);
    if (s == 1 || cost[s] < least) least = cost[s];
  }
  for (int s = 1; s <= 16; ++s)
    if (cost[s] > 0.0 && cost[s] <= 1.03 * least) return s;
  return 1;
}

// parts[run][rows, H] (fp32, runs `stride` elements apart) of dlogits[rows, V] W[V, H]
int dhidden_parts(const Head& h, const void* dlogits, float* parts, int64_t rows, int64_t stride, int runs,
                  const float* row_scale) {
  gemm::Launch L;
  L.dtype = h.dtype;
  L.a0.ptr = dlogits, L.a0.kmajor = 1, L.a0.mn = rows, L.a0.k = h.V, L.a0.ld = h.ld_logits;
  L.b0.ptr = h.W, L.b0.kmajor = 0, L.b0.mn = h.H, L.b0.k = h.V, L.b0.ld = h.H;
  L.p.M = static_cast<int>(rows);
  L.p.N = static_cast<int>(h.H);
  L.p.status = h.status;
  L.p.out = parts;
  L.p.ldo = h.H;
  L.p.out_fp32 = 1;
  L.p.vec_ok = rows_aligned(parts, h.H, 4) && stride % 4 == 0;
  L.p.splits = runs;
  L.p.split_stride = stride;
  L.p.row_alpha = row_scale;
  return gemm::launch<gemm::EPI_PLAIN>(L, h.s);
}

// out = T(alpha * sum over runs), in the runs' order; four elements per thread and step.  alpha: null is 1.
template <typename T>
__global__ void __launch_bounds__(kThreads)
sum_runs_kernel(const float* __restrict__ parts, T* __restrict__ out, int64_t n4, int runs, int64_t stride4,
                const float* __restrict__ alpha) {
  grid_dependency_wait();
  const float a = alpha != nullptr ? __ldg(alpha) : 1.f;
  const float4* in = reinterpret_cast<const float4*>(parts);
  const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < n4; i += step) {
    float4 v = __ldcs(in + i);
    for (int r = 1; r < runs; ++r) {
      const float4 u = __ldcs(in + r * stride4 + i);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    v.x *= a, v.y *= a, v.z *= a, v.w *= a;
    if constexpr (sizeof(T) == 4) {
      reinterpret_cast<float4*>(out)[i] = v;
    } else {
      T o[4] = {Cvt<T>::from_f(v.x), Cvt<T>::from_f(v.y), Cvt<T>::from_f(v.z), Cvt<T>::from_f(v.w)};
      reinterpret_cast<uint2*>(out)[i] = *reinterpret_cast<const uint2*>(o);
    }
  }
}

int sum_runs(const float* parts, void* out, int64_t n, int runs, int64_t stride, const float* alpha, int dtype,
             cudaStream_t s) {
  const int64_t n4 = n / 4;  // rows are whole 16-byte vectors
  const dim3 grid(grid_for(ceil_div(n4, kThreads), 16)), block(kThreads);
  cudaError_t e;
  if (dtype == BT_BF16)
    e = launch_dependent(sum_runs_kernel<__nv_bfloat16>, grid, block, 0, s, parts, static_cast<__nv_bfloat16*>(out), n4,
                         runs, stride / 4, alpha);
  else if (dtype == BT_FP16)
    e = launch_dependent(sum_runs_kernel<__half>, grid, block, 0, s, parts, static_cast<__half*>(out), n4, runs,
                         stride / 4, alpha);
  else
    e = launch_dependent(sum_runs_kernel<float>, grid, block, 0, s, parts, static_cast<float*>(out), n4, runs,
                         stride / 4, alpha);
  BT_CHECK_LAUNCHED(e, "logp: sum of d hidden");
  return BT_OK;
}

// out[V, H] = alpha (dlogits^T x + addend), x dense
int dweight(const Head& h, const void* dlogits, const void* x, void* out, int64_t rows, int out_dtype,
            const float* addend, const float* alpha) {
  return bt_gemm(dlogits, x, out, h.V, h.H, rows, h.ld_logits, h.H, h.H, 0, 0, h.dtype, out_dtype, addend, h.H, alpha,
                 h.status, h.s);
}

int policy_dlogits(const Head& h, void* logits, const float* tile_stats, const float* lse, const int64_t* labels,
                   const float* coef, int64_t rows, const Exponents& ex) {
  const int64_t vec = 16 / esize(h.dtype);
  // enough CTAs for ~8 per SM: rows are split into column segments when there are few
  const int sms = sm_count();
  int64_t gx = rows < static_cast<int64_t>(sms) * 8 ? rows : static_cast<int64_t>(sms) * 8;
  int64_t gy = 1;
  const int64_t nvec = (h.V + vec - 1) / vec;
  while (gx * gy < static_cast<int64_t>(sms) * 4 && gy * 2 * kThreads <= nvec) gy *= 2;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), block(kThreads);
  const float2* ts = reinterpret_cast<const float2*>(tile_stats);
  cudaError_t e;
  if (h.dtype == BT_BF16)
    e = launch_dependent(policy_dlogits_kernel<__nv_bfloat16>, grid, block, 0, h.s, static_cast<__nv_bfloat16*>(logits),
                         ts, lse, labels, coef, rows, h.V, h.ld_logits, h.n_vt, ex);
  else if (h.dtype == BT_FP16)
    e = launch_dependent(policy_dlogits_kernel<__half>, grid, block, 0, h.s, static_cast<__half*>(logits), ts, lse,
                         labels, coef, rows, h.V, h.ld_logits, h.n_vt, ex);
  else
    e = launch_dependent(policy_dlogits_kernel<float>, grid, block, 0, h.s, static_cast<float*>(logits), ts, lse,
                         labels, coef, rows, h.V, h.ld_logits, h.n_vt, ex);
  BT_CHECK_LAUNCHED(e, "policy: dlogits");
  return BT_OK;
}

int fill_head(Head* h, const char* what, const void* W, int64_t rows, int64_t H, int64_t V, int64_t ld_hidden,
              const void* hidden, int64_t chunk, int64_t ignore_index, int dtype, int32_t* status, void* stream) {
  BT_CHECK_ARG(known(dtype), "%s: unknown dtype %d", what, dtype);
  BT_CHECK_ARG(rows >= 0 && rows <= 0x7fffffffll && H > 0 && H <= 0x7fffffffll && V > 0 && V <= 0x7fffffffll,
               "%s: bad extents rows=%lld H=%lld V=%lld", what, (long long)rows, (long long)H, (long long)V);
  BT_CHECK_ARG(chunk > 0, "%s: chunk must be positive", what);
  BT_CHECK_ARG(rows == 0 || (hidden != nullptr && W != nullptr), "%s: null pointer", what);
  BT_CHECK_ARG(rows == 0 || (rows_aligned(hidden, rows > 1 ? ld_hidden : H, esize(dtype)) &&
                             rows_aligned(W, H, esize(dtype)) && (rows == 1 || ld_hidden >= H)),
               "%s: rows must be 16-byte aligned", what);
  h->W = W, h->H = H, h->V = V, h->ignore_index = ignore_index;
  h->ld_logits = (V + 7) / 8 * 8;
  h->dtype = dtype;
  h->n_vt = static_cast<int>(bt_lce_num_vtiles(V));
  h->status = status;
  h->s = static_cast<cudaStream_t>(stream);
  return BT_OK;
}

const char* row_ptr(const void* base, int64_t row, int64_t ld, int dtype) {
  return static_cast<const char*>(base) + row * ld * esize(dtype);
}
int64_t even(int64_t n) { return (n + 1) / 2 * 2; }  // pairs of floats are read as float2

}  // namespace
}  // namespace bt

int bt_internal_set_wait_limit_logp(unsigned long long ns) {
  return bt::ptx::set_wait_limit_ns(ns) == cudaSuccess ? 0 : -1;
}

extern "C" int64_t bt_logp_fwd_ws_floats(int64_t chunk, int64_t V) {
  if (chunk < 0 || V <= 0) return 0;
  return chunk * bt_lce_num_vtiles(V) * 2 + chunk;
}

extern "C" int bt_logp_fwd(const void* hidden, const void* W, const int64_t* labels, float* logp, float* lse, float* ws,
                           int64_t rows, int64_t H, int64_t V, int64_t ld_hidden, int64_t chunk, int64_t ignore_index,
                           int dtype, int32_t* status, void* stream) {
  using namespace bt;
  Head h;
  if (int rc = fill_head(&h, "logp_fwd", W, rows, H, V, ld_hidden, hidden, chunk, ignore_index, dtype, status, stream))
    return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(labels && logp && ws, "logp_fwd: null pointer");
  BT_CHECK_ARG(aligned8(ws), "logp_fwd: ws must be 8-byte aligned");
  float* tile_stats = ws;
  float* tgt = ws + chunk * h.n_vt * 2;
  for (int64_t r = 0; r < rows; r += chunk) {
    const int64_t n = rows - r < chunk ? rows - r : chunk;
    if (int rc = stats(h, row_ptr(hidden, r, ld_hidden, dtype), labels + r, nullptr, tile_stats, tgt, n, ld_hidden))
      return rc;
    BT_CHECK_LAUNCHED(launch_dependent(logp_rows_kernel, dim3(grid_for(ceil_div(n, kThreads / 32), 8)), dim3(kThreads),
                                       0, h.s, reinterpret_cast<const float2*>(tile_stats), tgt, labels + r, logp + r,
                                       lse != nullptr ? lse + r : nullptr, n, h.n_vt, ignore_index, V, status),
                      "logp_fwd: rows");
  }
  return BT_OK;
}

extern "C" int bt_logp_bwd(const float* dlogp, const void* hidden, const void* W, const int64_t* labels,
                           const float* lse, void* masked, void* dlogits, void* dhidden, float* dhidden_parts_,
                           void* dweight_out, float* dweight_acc, float* ws, int64_t rows, int64_t H, int64_t V,
                           int64_t ld_hidden, int64_t chunk, int64_t ignore_index, int dtype, int dweight_dtype,
                           int32_t* status, void* stream) {
  using namespace bt;
  Head h;
  if (int rc = fill_head(&h, "logp_bwd", W, rows, H, V, ld_hidden, hidden, chunk, ignore_index, dtype, status, stream))
    return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(dlogp && labels && lse && masked && dlogits && ws, "logp_bwd: null pointer");
  BT_CHECK_ARG(aligned16(masked) && aligned16(dlogits), "logp_bwd: buffers must be 16-byte aligned");
  BT_CHECK_ARG(dhidden == nullptr || (dhidden_parts_ != nullptr && aligned16(dhidden) && aligned16(dhidden_parts_)),
               "logp_bwd: the gradient of hidden needs 16-byte aligned buffers for itself and its parts");
  BT_CHECK_ARG(dweight_out == nullptr || rows <= chunk || dweight_acc != nullptr,
               "logp_bwd: more than one chunk needs an accumulator for the weight gradient");
  if (chunk > rows) chunk = rows;
  const int runs = dhidden_runs(chunk, H, V, dtype);
  float* scal = ws;  // [1 + 2 rows]: scale back, coefficients, fp16's scales of the rows
  float* coef = ws + 1;
  float* row_scale = dtype == BT_FP16 ? coef + rows : nullptr;
  BT_CHECK_LAUNCHED(launch_dependent(logp_coef_kernel, dim3(1), dim3(1024), 0, h.s, dlogp, labels, rows, ignore_index,
                                     V, coef, row_scale, scal),
                    "logp_bwd: coefficients");
  const int64_t ld = rows > 1 ? ld_hidden : H;
  if (int rc = mask_rows(h, hidden, masked, labels, rows, ld, nullptr, nullptr, 0, row_scale)) return rc;
  for (int64_t r = 0; r < rows; r += chunk) {
    const int64_t n = rows - r < chunk ? rows - r : chunk;
    const char* x = row_ptr(masked, r, H, dtype);
    // (logits of ignored rows, which may be anything, are never used; `masked` is for the weight's product)
    gemm::Launch L = head_product(h, row_ptr(hidden, r, ld, dtype), labels + r, n, ld);
    L.p.row_lse = lse + r;
    L.p.row_coef = coef + r;
    L.p.out = dlogits;
    L.p.ldo = h.ld_logits;
    L.p.vec_ok = rows_aligned(dlogits, h.ld_logits, esize(dtype));
    if (int rc = gemm::launch<gemm::EPI_DLOGITS>(L, h.s)) return rc;
    if (dhidden != nullptr) {
      if (int rc = dhidden_parts(h, dlogits, dhidden_parts_, n, chunk * H, runs,
                                 row_scale != nullptr ? row_scale + r : nullptr))
        return rc;
      if (int rc = sum_runs(dhidden_parts_, const_cast<char*>(row_ptr(dhidden, r, H, dtype)), n * H, runs, chunk * H,
                            scal, dtype, h.s))
        return rc;
    }
    if (dweight_out != nullptr) {
      const bool last = r + n == rows;
      if (int rc = dweight(h, dlogits, x, last ? dweight_out : dweight_acc, n, last ? dweight_dtype : BT_FP32,
                           r > 0 ? dweight_acc : nullptr, last ? scal : nullptr))
        return rc;
    }
  }
  return BT_OK;
}

extern "C" int64_t bt_dhidden_runs(int64_t rows, int64_t H, int64_t V, int dtype) {
  using namespace bt;
  return rows > 0 && H > 0 && V > 0 && known(dtype) ? dhidden_runs(rows, H, V, dtype) : 1;
}

extern "C" int bt_sum_runs(const float* parts, void* out, int64_t n, int64_t runs, int64_t stride, const float* alpha,
                           int dtype, void* stream) {
  using namespace bt;
  BT_CHECK_ARG(known(dtype), "sum_runs: unknown dtype %d", dtype);
  BT_CHECK_ARG(n >= 0 && n % 4 == 0 && runs >= 1 && runs <= 1024 && (runs == 1 || (stride >= n && stride % 4 == 0)),
               "sum_runs: bad sizes");
  if (n == 0) return BT_OK;
  BT_CHECK_ARG(parts && out && alpha, "sum_runs: null pointer");
  BT_CHECK_ARG(aligned16(parts) && aligned16(out), "sum_runs: buffers must be 16-byte aligned");
  return sum_runs(parts, out, n, static_cast<int>(runs), stride, alpha, dtype, static_cast<cudaStream_t>(stream));
}

extern "C" int64_t bt_policy_fwd_ws_floats(int64_t rows, int64_t chunk, int64_t n_seq, int64_t V) {
  if (rows < 0 || chunk < 0 || n_seq < 0 || V <= 0) return 0;
  return bt::even(n_seq + 3 * rows + 3 * chunk) + chunk * bt_lce_num_vtiles(V) * 2;
}

extern "C" int bt_policy_fwd(const bt_policy_desc* d, int32_t* status, void* stream) {
  using namespace bt;
  BT_CHECK_ARG(d != nullptr, "policy_fwd: null descriptor");
  Head h;
  if (int rc = fill_head(&h, "policy_fwd", d->W, d->rows, d->H, d->V, d->ld_hidden, d->hidden, d->chunk,
                         d->ignore_index, d->dtype, status, stream))
    return rc;
  BT_CHECK_ARG(d->n_seq >= 0 && d->n_seq < (1 << 24) && (d->cu_seqlens != nullptr || d->n_seq == 1),
               "policy_fwd: bad sequence count");
  BT_CHECK_ARG(d->ws && d->loss && d->averages, "policy_fwd: null pointer");
  BT_CHECK_ARG(aligned8(d->ws), "policy_fwd: ws must be 8-byte aligned");
  const bool grad = d->dhidden != nullptr || d->want_dweight != 0;
  if (d->rows > 0) {
    BT_CHECK_ARG(d->labels && d->old_logp && d->adv && d->logp, "policy_fwd: null pointer");
    BT_CHECK_ARG(!grad || (d->masked && d->logits && aligned16(d->masked) && aligned16(d->logits)),
                 "policy_fwd: gradients need 16-byte aligned buffers for the counted rows and the logits");
    BT_CHECK_ARG(!d->want_dweight || d->rows <= d->chunk || (d->dweight_acc != nullptr && aligned16(d->dweight_acc)),
                 "policy_fwd: more than one chunk needs a 16-byte aligned accumulator for the weight gradient");
  }
  const int runs = d->rows > 0 ? dhidden_runs(d->chunk < d->rows ? d->chunk : d->rows, d->H, d->V, d->dtype) : 1;
  // one chunk: its runs are added up when the upstream gradient is known; more: each before the next
  const bool sum_now = d->rows > d->chunk && runs > 1;
  BT_CHECK_ARG(d->dhidden == nullptr || !sum_now ||
                   (d->dhidden_parts != nullptr && aligned16(d->dhidden_parts) && aligned16(d->dhidden)),
               "policy_fwd: more than one chunk needs 16-byte aligned buffers for the gradient of hidden and its parts");
  float* scal = d->averages + 2;
  // E after chunk k is word k % 3: the one before it is still needed beside it, and the next is prepared
  int32_t* top_exp = reinterpret_cast<int32_t*>(d->averages + 5);
  const bool scaled = grad && d->dtype == BT_FP16;
  float* weights = d->ws;
  float* terms = weights + d->n_seq;
  float* lse = terms + 3 * d->rows;
  float* coef = lse + d->chunk;
  float* tgt = coef + d->chunk;
  float* tile_stats = d->ws + even(d->n_seq + 3 * d->rows + 3 * d->chunk);
  BT_CHECK_LAUNCHED(launch_dependent(policy_weights_kernel, dim3(1), dim3(1024), 0, h.s, d->labels, d->rows,
                                     d->cu_seqlens, static_cast<int>(d->n_seq), d->ignore_index, d->V, weights, scal,
                                     top_exp, status),
                    "policy_fwd: weights");
  const void* x = d->hidden;
  int64_t ld_x = d->ld_hidden;
  if (grad && d->rows > 0) {
    if (int rc = mask_rows(h, d->hidden, d->masked, d->labels, d->rows, d->rows > 1 ? d->ld_hidden : d->H, scal,
                           d->cu_seqlens, static_cast<int>(d->n_seq), nullptr))
      return rc;
    x = d->masked;
    ld_x = d->H;
  }
  int k = 0;  // chunk
  for (int64_t r = 0; r < d->rows; r += d->chunk, ++k) {
    const int64_t n = d->rows - r < d->chunk ? d->rows - r : d->chunk;
    const char* xc = row_ptr(x, r, ld_x, d->dtype);
    if (int rc = stats(h, xc, d->labels + r, grad ? d->logits : nullptr, tile_stats, tgt, n, ld_x)) return rc;
    PolicyArgs a{};
    a.tile_stats = reinterpret_cast<const float2*>(tile_stats);
    a.tgt_logit = tgt, a.labels = d->labels + r, a.old_logp = d->old_logp, a.adv = d->adv, a.ref_logp = d->ref_logp;
    a.cu = d->cu_seqlens, a.weights = weights, a.scal = scal, a.logp = d->logp + r, a.lse = lse, a.coef = coef;
    a.terms = terms, a.rows = n, a.row0 = r, a.total = d->rows, a.ignore_index = d->ignore_index, a.vocab = d->V;
    a.n_vt = h.n_vt, a.n_seq = static_cast<int>(d->n_seq);
    a.row_scale = scaled ? tgt : nullptr, a.top_exp = top_exp + k % 3;
    a.clip_low = d->clip_low, a.clip_high = d->clip_high, a.kl_coef = d->kl_coef;
    BT_CHECK_LAUNCHED(launch_dependent(policy_rows_kernel, dim3(grid_for(ceil_div(n, kThreads / 32), 8)),
                                       dim3(kThreads), 0, h.s, a),
                      "policy_fwd: rows");
    if (!grad) continue;
    const Exponents ex{a.row_scale, a.top_exp, top_exp + (k + 1) % 3, const_cast<char*>(xc), d->H};
    if (int rc = policy_dlogits(h, d->logits, tile_stats, lse, d->labels + r, coef, n, ex)) return rc;
    if (d->dhidden != nullptr) {
      float* sum = d->dhidden + r * d->H;
      if (int rc = dhidden_parts(h, d->logits, sum_now ? d->dhidden_parts : sum, n,
                                 (sum_now ? d->chunk : d->rows) * d->H, runs, a.row_scale))
        return rc;
      if (sum_now) {
        if (int rc = sum_runs(d->dhidden_parts, sum, n * d->H, runs, d->chunk * d->H, nullptr, BT_FP32, h.s)) return rc;
      }
    }
    if (scaled && d->want_dweight && r > 0) {
      const int64_t n4 = d->V * d->H / 4;
      BT_CHECK_LAUNCHED(launch_dependent(policy_rescale_kernel, dim3(grid_for(ceil_div(n4, kThreads), 16)),
                                         dim3(kThreads), 0, h.s, d->dweight_acc, n4, top_exp + (k + 2) % 3, a.top_exp),
                        "policy_fwd: sum of d weight");
    }
    if (d->want_dweight && r + n < d->rows) {  // the last chunk's product waits for the upstream gradient
      if (int rc = dweight(h, d->logits, xc, d->dweight_acc, n, BT_FP32, r > 0 ? d->dweight_acc : nullptr, nullptr))
        return rc;
    }
  }
  BT_CHECK_LAUNCHED(launch_dependent(policy_reduce_kernel, dim3(3), dim3(1024), 0, h.s, terms, d->rows, d->loss,
                                     d->averages, scaled && k > 0 ? top_exp + (k - 1) % 3 : nullptr),
                    "policy_fwd: sums");
  return BT_OK;
}
