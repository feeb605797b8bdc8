// Log-probabilities of tokens through the output head and the clipped policy loss on them: the
// logits products (tcgen05 GEMM core) with their epilogues, and the row kernels between them.
//
//   logp_t = logit_t[y_t] - lse_t                      d logp_t / d logit_t = onehot(y_t) - softmax
//   r_t = exp(logp_t - old_t)
//   loss = sum_t w_t ( -min(r_t A_t, clip(r_t, 1 - lo, 1 + hi) A_t) + kl_coef (e^d - d - 1) ),  d = ref_t - logp_t
//   w_t = 1 / tokens, or 1 / (sequences * tokens of t's sequence)
#include "gemm_sm100.cuh"

namespace bt {
namespace {

constexpr int kThreads = 256;

bool rows_aligned(const void* p, int64_t ld, int elem_bytes) {
  return p != nullptr && aligned16(p) && (ld * elem_bytes) % 16 == 0;
}
bool known(int dtype) { return dtype == BT_BF16 || dtype == BT_FP16 || dtype == BT_FP32; }
int esize(int dtype) { return dtype == BT_FP32 ? 4 : 2; }
int check_sizes(const char* what, int64_t rows, int64_t h, int64_t v, int dtype) {
  BT_CHECK_ARG(known(dtype), "%s: unknown dtype %d", what, dtype);
  BT_CHECK_ARG(rows >= 0 && rows <= 0x7fffffffll && h > 0 && h <= 0x7fffffffll && v > 0 && v <= 0x7fffffffll,
               "%s: bad extents rows=%lld H=%lld V=%lld", what, (long long)rows, (long long)h, (long long)v);
  return BT_OK;
}

__device__ __forceinline__ bool counted(int64_t label, int64_t ignore_index, int64_t vocab) {
  return label != ignore_index && label >= 0 && label < vocab;
}

// (max, sum exp) of a row from its half tiles; all lanes of the warp get the result.
__device__ __forceinline__ float2 merge_stats(const float2* __restrict__ ts, int n_vt, int lane) {
  float mx = -1e30f, sum = 0.f;
  for (int i = lane; i < n_vt; i += 32) {
    const float2 t = ts[i];
    const float nm = fmaxf(mx, t.x);
    sum = sum * __expf(mx - nm) + t.y * __expf(t.x - nm);
    mx = nm;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float omx = __shfl_xor_sync(0xffffffffu, mx, o);
    const float osum = __shfl_xor_sync(0xffffffffu, sum, o);
    const float nm = fmaxf(mx, omx);
    sum = sum * __expf(mx - nm) + osum * __expf(omx - nm);
    mx = nm;
  }
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

// Upstream gradient of the log-probabilities as the coefficients of the dlogits product, scaled by a
// power of two so that the largest is in [1/2, 1): with fp16 operands a mean over many tokens would
// otherwise push them, times the softmax, below the type's range.  scal[0] = scale back.
__global__ void __launch_bounds__(1024)
logp_coef_kernel(const float* __restrict__ dlogp, const int64_t* __restrict__ labels, int64_t n, int64_t ignore_index,
                 int64_t vocab, float* __restrict__ coef, float* __restrict__ scal) {
  grid_dependency_wait();
  __shared__ float s_max[32];
  float mx = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += 1024)
    if (counted(labels[i], ignore_index, vocab)) {
      const float a = fabsf(dlogp[i]);
      if (a <= 3.0e38f) mx = fmaxf(mx, a);  // infinities and NaN keep their place, but set no scale
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
  for (int64_t i = threadIdx.x; i < n; i += 1024)
    coef[i] = counted(labels[i], ignore_index, vocab) ? dlogp[i] * up : 0.f;
}

// Rows of `x` that count, copied; zeros in the place of the others, which meet zero coefficients in
// the weight gradient's product and must be finite there.
template <typename T>
__global__ void __launch_bounds__(kThreads)
logp_mask_rows_kernel(const T* __restrict__ x, T* __restrict__ y, const int64_t* __restrict__ labels, int64_t rows,
                      int64_t h, int64_t ld, int64_t ignore_index, int64_t vocab) {
  grid_dependency_wait();
  constexpr int E = Cvt<T>::N;
  const int64_t nvec = h / E;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const bool in = counted(labels[row], ignore_index, vocab);
    for (int64_t i = threadIdx.x; i < nvec; i += kThreads)
      st_global_v4(y + row * h + i * E, in ? ld_stream_v4(x + row * ld + i * E) : make_uint4(0, 0, 0, 0));
  }
}

// ------------------------------------------------------------------ the policy loss
// Weight of a counted token of each sequence (one entry for all tokens without offsets), and
// scal[0] = largest weight, scal[1] = 1 / that: coefficients are stored relative to it.
__global__ void __launch_bounds__(1024)
policy_weights_kernel(const int64_t* __restrict__ labels, int64_t n, const int32_t* __restrict__ cu, int n_seq,
                      int64_t ignore_index, int64_t vocab, float* __restrict__ weights, float* __restrict__ scal,
                      int32_t* __restrict__ status) {
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
    scal[1] = static_cast<float>(1.0 / top);
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
  float* terms;  // [3][total]: weighted loss, kl, clipped
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
        term += a.kl_coef * kl;
        coef -= a.kl_coef * em1;
      }
    }
    a.logp[row] = static_cast<float>(logp);
    a.lse[row] = st.x + logf(st.y);
    a.coef[row] = static_cast<float>(coef * w * static_cast<double>(a.scal[1]));
    a.terms[g] = static_cast<float>(term * w);
    a.terms[a.total + g] = static_cast<float>(kl * w);
    a.terms[2 * a.total + g] = held ? w : 0.f;
  }
}

// out[0..2] = sums of the three rows of terms (fp64, fixed order).
__global__ void __launch_bounds__(1024)
policy_reduce_kernel(const float* __restrict__ terms, int64_t n, float* __restrict__ out) {
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
    out[blockIdx.x] = static_cast<float>(s);
  }
}

// Shifted logits -> coef (onehot - softmax), in place: one read and one write of the chunk, 16 bytes
// per thread and step.  exp(logit - lse) = exp(stored) exp(half-tile max - lse), the second factor
// once per vector.
template <typename T>
__global__ void __launch_bounds__(kThreads)
policy_dlogits_kernel(T* __restrict__ logits, const float2* __restrict__ tile_stats, const float* __restrict__ lse,
                      const int64_t* __restrict__ labels, const float* __restrict__ coef, int64_t rows, int64_t V,
                      int64_t ld, int n_vt) {
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
}

unsigned grid_for(int64_t blocks, int per_sm) {
  const int64_t cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<unsigned>(blocks < 1 ? 1 : (blocks < cap ? blocks : cap));
}

gemm::Launch head_product(const void* hidden, const void* W, const int64_t* labels, int64_t rows, int64_t H, int64_t V,
                          int64_t ld_hidden, int64_t ignore_index, int dtype, int32_t* status) {
  gemm::Launch L;
  L.dtype = dtype;
  L.a0.ptr = hidden, L.a0.kmajor = 1, L.a0.mn = rows, L.a0.k = H, L.a0.ld = ld_hidden;
  L.b0.ptr = W, L.b0.kmajor = 1, L.b0.mn = V, L.b0.k = H, L.b0.ld = H;
  L.p.M = static_cast<int>(rows);
  L.p.N = static_cast<int>(V);
  L.p.status = status;
  L.p.labels = labels;
  L.p.ignore_index = ignore_index;
  L.p.n_vtiles = static_cast<int>(bt_lce_num_vtiles(V));
  return L;
}

}  // namespace
}  // namespace bt

int bt_internal_set_wait_limit_logp(unsigned long long ns) {
  return bt::ptx::set_wait_limit_ns(ns) == cudaSuccess ? 0 : -1;
}

extern "C" int bt_logp_stats(const void* hidden, const void* W, const int64_t* labels, void* logits, float* tile_stats,
                             float* tgt_logit, int64_t rows, int64_t H, int64_t V, int64_t ld_hidden, int64_t ld_logits,
                             int64_t ignore_index, int dtype, int32_t* status, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("logp_stats", rows, H, V, dtype)) return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(hidden && W && labels && tile_stats && tgt_logit, "logp_stats: null pointer");
  BT_CHECK_ARG(logits == nullptr || ld_logits >= V, "logp_stats: logits stride smaller than V");
  gemm::Launch L = head_product(hidden, W, labels, rows, H, V, ld_hidden, ignore_index, dtype, status);
  L.p.tile_stats = tile_stats;
  L.p.tgt_logit = tgt_logit;
  if (logits == nullptr) return gemm::launch<gemm::EPI_LOGP>(L, static_cast<cudaStream_t>(stream));
  L.p.out = logits;
  L.p.ldo = ld_logits;
  L.p.vec_ok = rows_aligned(logits, ld_logits, esize(dtype));
  return gemm::launch<gemm::EPI_LOGP_SHIFT>(L, static_cast<cudaStream_t>(stream));
}

extern "C" int bt_logp_dlogits(const void* hidden, const void* W, const int64_t* labels, const float* lse,
                               const float* coef, void* dlogits, int64_t rows, int64_t H, int64_t V, int64_t ld_hidden,
                               int64_t ld_dlogits, int dtype, int32_t* status, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("logp_dlogits", rows, H, V, dtype)) return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(hidden && W && labels && lse && coef && dlogits, "logp_dlogits: null pointer");
  BT_CHECK_ARG(ld_dlogits >= V, "logp_dlogits: dlogits stride smaller than V");
  gemm::Launch L = head_product(hidden, W, labels, rows, H, V, ld_hidden, 0, dtype, status);
  L.p.row_lse = lse;
  L.p.row_coef = coef;
  L.p.out = dlogits;
  L.p.ldo = ld_dlogits;
  L.p.vec_ok = rows_aligned(dlogits, ld_dlogits, esize(dtype));
  return gemm::launch<gemm::EPI_DLOGITS>(L, static_cast<cudaStream_t>(stream));
}

extern "C" int bt_logp_rows(const float* tile_stats, const float* tgt_logit, const int64_t* labels, float* logp,
                            float* lse, int64_t rows, int64_t V, int64_t ignore_index, int32_t* status, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("logp_rows", rows, 1, V, BT_BF16)) return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(tile_stats && tgt_logit && labels && logp, "logp_rows: null pointer");
  BT_CHECK_LAUNCHED(launch_dependent(logp_rows_kernel, dim3(grid_for(ceil_div(rows, kThreads / 32), 8)), dim3(kThreads),
                                     0, static_cast<cudaStream_t>(stream), reinterpret_cast<const float2*>(tile_stats),
                                     tgt_logit, labels, logp, lse, rows, static_cast<int>(bt_lce_num_vtiles(V)),
                                     ignore_index, V, status),
                    "logp_rows");
  return BT_OK;
}

extern "C" int bt_logp_coef(const float* dlogp, const int64_t* labels, int64_t n, int64_t V, int64_t ignore_index,
                            float* coef, float* scal, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("logp_coef", n, 1, V, BT_BF16)) return rc;
  BT_CHECK_ARG(scal && (n == 0 || (dlogp && labels && coef)), "logp_coef: null pointer");
  BT_CHECK_LAUNCHED(launch_dependent(logp_coef_kernel, dim3(1), dim3(1024), 0, static_cast<cudaStream_t>(stream), dlogp,
                                     labels, n, ignore_index, V, coef, scal),
                    "logp_coef");
  return BT_OK;
}

extern "C" int bt_logp_mask_rows(const void* x, void* y, const int64_t* labels, int64_t rows, int64_t H, int64_t ld,
                                 int64_t V, int64_t ignore_index, int dtype, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("logp_mask_rows", rows, H, V, dtype)) return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(x && y && labels, "logp_mask_rows: null pointer");
  BT_CHECK_ARG(rows_aligned(x, ld, esize(dtype)) && rows_aligned(y, H, esize(dtype)) && (rows == 1 || ld >= H),
               "logp_mask_rows: rows must be 16-byte aligned");
  const dim3 grid(grid_for(rows, 8)), block(kThreads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BT_FP32)
    BT_CHECK_LAUNCHED(launch_dependent(logp_mask_rows_kernel<float>, grid, block, 0, s, static_cast<const float*>(x),
                                       static_cast<float*>(y), labels, rows, H, ld, ignore_index, V),
                      "logp_mask_rows");
  else  // a copy: the two 16-bit types are the same
    BT_CHECK_LAUNCHED(launch_dependent(logp_mask_rows_kernel<__half>, grid, block, 0, s, static_cast<const __half*>(x),
                                       static_cast<__half*>(y), labels, rows, H, ld, ignore_index, V),
                      "logp_mask_rows");
  return BT_OK;
}

extern "C" int bt_policy_weights(const int64_t* labels, int64_t n, const int32_t* cu_seqlens, int64_t n_seq, int64_t V,
                                 int64_t ignore_index, float* weights, float* scal, int32_t* status, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("policy_weights", n, 1, V, BT_BF16)) return rc;
  BT_CHECK_ARG(n_seq >= 0 && n_seq < (1 << 24) && (cu_seqlens != nullptr || n_seq == 1), "policy_weights: bad sequence count");
  BT_CHECK_ARG(weights && scal && (n == 0 || labels), "policy_weights: null pointer");
  BT_CHECK_LAUNCHED(launch_dependent(policy_weights_kernel, dim3(1), dim3(1024), 0, static_cast<cudaStream_t>(stream),
                                     labels, n, cu_seqlens, static_cast<int>(n_seq), ignore_index, V, weights, scal,
                                     status),
                    "policy_weights");
  return BT_OK;
}

extern "C" int bt_policy_rows(const float* tile_stats, const float* tgt_logit, const int64_t* labels,
                              const float* old_logp, const float* adv, const float* ref_logp, const int32_t* cu_seqlens,
                              const float* weights, const float* scal, float* logp, float* lse, float* coef,
                              float* terms, int64_t rows, int64_t row0, int64_t total, int64_t n_seq, int64_t V,
                              int64_t ignore_index, float clip_low, float clip_high, float kl_coef, void* stream) {
  using namespace bt;
  if (int rc = check_sizes("policy_rows", total, 1, V, BT_BF16)) return rc;
  BT_CHECK_ARG(rows >= 0 && row0 >= 0 && row0 + rows <= total, "policy_rows: chunk outside the batch");
  BT_CHECK_ARG(n_seq >= 0 && n_seq < (1 << 24) && (cu_seqlens != nullptr || n_seq == 1), "policy_rows: bad sequence count");
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(tile_stats && tgt_logit && labels && old_logp && adv && weights && scal && logp && lse && coef && terms,
               "policy_rows: null pointer");
  PolicyArgs a{};
  a.tile_stats = reinterpret_cast<const float2*>(tile_stats);
  a.tgt_logit = tgt_logit, a.labels = labels, a.old_logp = old_logp, a.adv = adv, a.ref_logp = ref_logp;
  a.cu = cu_seqlens, a.weights = weights, a.scal = scal, a.logp = logp, a.lse = lse, a.coef = coef, a.terms = terms;
  a.rows = rows, a.row0 = row0, a.total = total, a.ignore_index = ignore_index, a.vocab = V;
  a.n_vt = static_cast<int>(bt_lce_num_vtiles(V)), a.n_seq = static_cast<int>(n_seq);
  a.clip_low = clip_low, a.clip_high = clip_high, a.kl_coef = kl_coef;
  BT_CHECK_LAUNCHED(launch_dependent(policy_rows_kernel, dim3(grid_for(ceil_div(rows, kThreads / 32), 8)),
                                     dim3(kThreads), 0, static_cast<cudaStream_t>(stream), a),
                    "policy_rows");
  return BT_OK;
}

extern "C" int bt_policy_dlogits(void* logits, const float* tile_stats, const float* lse, const int64_t* labels,
                                 const float* coef, int64_t rows, int64_t V, int64_t ld_logits, int dtype,
                                 void* stream) {
  using namespace bt;
  if (int rc = check_sizes("policy_dlogits", rows, 1, V, dtype)) return rc;
  if (rows == 0) return BT_OK;
  BT_CHECK_ARG(logits && tile_stats && lse && labels && coef, "policy_dlogits: null pointer");
  const int64_t vec = 16 / esize(dtype);
  BT_CHECK_ARG(rows_aligned(logits, ld_logits, esize(dtype)) && ld_logits >= (V + vec - 1) / vec * vec,
               "policy_dlogits: logits rows must be 16-byte aligned and padded to whole 16-byte vectors");
  const int sms = sm_count();
  int64_t gx = rows < static_cast<int64_t>(sms) * 8 ? rows : static_cast<int64_t>(sms) * 8;
  int64_t gy = 1;
  const int64_t nvec = (V + vec - 1) / vec;
  while (gx * gy < static_cast<int64_t>(sms) * 4 && gy * 2 * kThreads <= nvec) gy *= 2;
  const dim3 grid(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), block(kThreads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const float2* ts = reinterpret_cast<const float2*>(tile_stats);
  const int n_vt = static_cast<int>(bt_lce_num_vtiles(V));
  cudaError_t e;
  if (dtype == BT_BF16)
    e = launch_dependent(policy_dlogits_kernel<__nv_bfloat16>, grid, block, 0, s, static_cast<__nv_bfloat16*>(logits),
                         ts, lse, labels, coef, rows, V, ld_logits, n_vt);
  else if (dtype == BT_FP16)
    e = launch_dependent(policy_dlogits_kernel<__half>, grid, block, 0, s, static_cast<__half*>(logits), ts, lse,
                         labels, coef, rows, V, ld_logits, n_vt);
  else
    e = launch_dependent(policy_dlogits_kernel<float>, grid, block, 0, s, static_cast<float*>(logits), ts, lse, labels,
                         coef, rows, V, ld_logits, n_vt);
  BT_CHECK_LAUNCHED(e, "policy_dlogits");
  return BT_OK;
}

extern "C" int bt_policy_reduce(const float* terms, int64_t n, float* out, void* stream) {
  using namespace bt;
  BT_CHECK_ARG(n >= 0 && out && (n == 0 || terms), "policy_reduce: bad args");
  BT_CHECK_LAUNCHED(launch_dependent(policy_reduce_kernel, dim3(3), dim3(1024), 0, static_cast<cudaStream_t>(stream),
                                     terms, n, out),
                    "policy_reduce");
  return BT_OK;
}
