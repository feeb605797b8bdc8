// Causal attention over packed sequences, forward, and the plan that all attention kernels share.
//
//   O_i = sum_{j <= i} P_ij V_j,   P_ij = exp(scale q_i.k_j - lse_i),   i, j in the same sequence
//
// One CTA per (query tile of 128 packed rows, key/value head), two CTAs on an SM: 256 threads,
//   warps 0..3  softmax, one row per thread, and the epilogue
//   warp 4      issues tcgen05.mma:  S = Q K_j^T,  O += P_j V_j
//   warp 5      TMA loads: Q once, then K_0, V_0, K_1, ... (one tile of each at a time)
// (warps 6, 7 complete the warpgroup that hands its registers to the softmax warps).
// Tensor memory (256 columns): S (fp32, 128 columns; the 16-bit P replaces the first half and is the A
// operand of the second product) and O.  A key block takes a CTA about 3600 cycles - scores, softmax,
// second product - of which its products are 1050 and its exponentials 1024: the other CTA's products
// and exponentials run meanwhile, and under its start and its end as well, which no second tile inside
// one CTA can do.  Against two tiles per CTA and one CTA per SM (bf16, 32 / 8 heads of 128): 861 -> 830
// thousand cycles on one sequence of 8192 tokens, 69 -> 60 us on a ragged batch of 4096.
// Measured: 8192 tokens 457 us (468 with the residual stored), 1.20 PFLOP/s of the products executed (masked
// halves of the diagonal tiles included); at 4096 the matrix pipe is busy in 48% of the cycles and the
// exponentials' in 50%, the rest is the hand-over between them.  Exponentials on the FMA pipes instead took
// fewer cycles and the same time: what is left is the chip's power limit.
#include <mutex>

#include "attn_sm100.cuh"

namespace bt {
namespace attn {
namespace {

// ------------------------------------------------------------------ the plan
constexpr int kPlanThreads = 1024;

__global__ void __launch_bounds__(kPlanThreads)
attn_plan_kernel(const int32_t* __restrict__ cu, int batch, int total, int32_t* __restrict__ words,
                 int32_t* __restrict__ status) {
  grid_dependency_wait();
  __shared__ int s_len[kPlanSort];
  __shared__ unsigned long long s_area;  // below 2^61: the lengths sum to less than 2^30
  __shared__ int s_longest;
  const int tid = threadIdx.x;
  const int n = batch + 1;
  int32_t* start = words;
  int32_t* len = words + n;
  // offsets have to start at 0, never fall, and end within the tensor; anything else is reported and
  // read as "no sequence at all", so that no kernel that follows the plan can leave the tensors
  bool bad = false;
  unsigned long long area = 0;
  int longest = 0;
  if (tid == 0) s_area = 0, s_longest = 0;
  for (int i = tid; i < batch; i += kPlanThreads) {
    const int a = cu[i], b = cu[i + 1];
    const bool wrong = a < 0 || b < a || b > total || (i == 0 && a != 0);
    bad |= wrong;
    if (!wrong) {
      area += static_cast<unsigned long long>(b - a) * (b - a + kTile);
      longest = max(longest, b - a);
    }
  }
  bad = __syncthreads_or(bad);
  if (!bad && (tid & ~31) < batch) {  // warps that have seen a sequence
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) area += __shfl_xor_sync(0xffffffffu, area, o);
    longest = __reduce_max_sync(0xffffffffu, longest);
    if ((tid & 31) == 0) {
      atomicAdd(&s_area, area);
      atomicMax(&s_longest, longest);
    }
  }
  if (bad && tid == 0 && status != nullptr) atomicOr(status, BT_STATUS_BAD_SEQUENCES);
  if (batch <= kPlanSort) {
    // longest first: the tiles of a launch are started in plan order, so the last ones are small
    if (tid < batch) s_len[tid] = bad ? 0 : cu[tid + 1] - cu[tid];
    __syncthreads();
    if (tid < batch) {
      const int mine = s_len[tid];
      int rank = 0;
      for (int j = 0; j < batch; ++j) rank += s_len[j] > mine || (s_len[j] == mine && j < tid);
      start[rank] = bad ? 0 : cu[tid];
      len[rank] = mine;
    }
  } else {
    for (int i = tid; i < batch; i += kPlanThreads) {
      start[i] = bad ? 0 : cu[i];
      len[i] = bad ? 0 : cu[i + 1] - cu[i];
    }
  }
  if (tid == 0) {
    const int covered = (bad || batch == 0) ? 0 : cu[batch];
    start[batch] = covered;
    len[batch] = total - covered;
  }
  __syncthreads();
  if (tid == 0) {
    words[2 * n + kGrans * (n + 1)] = __float_as_int(static_cast<float>(s_area));
    words[2 * n + kGrans * (n + 1) + 1] = s_longest;
  }
  const int g = tid >> 5, lane = tid & 31;
  if (g < kGrans) {  // one warp per tile height: running tile counts
    int32_t* pre = words + 2 * n + g * (n + 1);
    int run = 0;
    for (int i0 = 0; i0 < n; i0 += 32) {
      const int i = i0 + lane;
      int c = i < n ? (len[i] + gran_of(g) - 1) / gran_of(g) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, c, o);
        if (lane >= o) c += up;
      }
      if (i < n) pre[i + 1] = run + c;
      run += __shfl_sync(0xffffffffu, c, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
}

// --------------------------------------------------------------- the forward
constexpr int kFwdThreads = 256;

template <int DT>
struct FwdGeo {
  static constexpr int kTileBytes = (DT / 64) * kBoxBytes;
  static constexpr int kSmem = 3 * kTileBytes + 512;  // Q, K, V and the barriers: two CTAs fit an SM
};

// Rescaling the output accumulator is put off until a row's maximum has grown by more than this many
// powers of two: P then stays below 2^8, far inside both 16-bit types, and the sums stay fp32.
constexpr float kLazyMax = 8.0f;

template <typename T, int DT>
__global__ void __launch_bounds__(kFwdThreads, 2)
attn_fwd_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmO,
                const __grid_constant__ CUtensorMap tmL, const Params p) {
  using G = FwdGeo<DT>;
  constexpr int TB = G::kTileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (!aligned_start(smem, p.status)) return;
  const uint32_t sQ = ptx::smem_u32(smem), sK = sQ + TB, sV = sK + TB;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + 3 * TB);
  uint64_t* k_full = q_full + 1;
  uint64_t* v_full = k_full + 1;
  uint64_t* s_full = v_full + 1;   // phase j: scores j are there, and K_j may be replaced
  uint64_t* p_ready = s_full + 1;
  uint64_t* pv_done = p_ready + 1; // phase j: block j is in O, and V_j may be replaced
  uint64_t* staged = pv_done + 1;
  uint64_t* fix = staged + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fix + 1);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(k_full, 1);
    ptx::mbar_init(v_full, 1);
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(p_ready, 4);
    ptx::mbar_init(pv_done, 1);
    ptx::mbar_init(staged, 4);
    ptx::mbar_init(fix, 1);
    *cta_abort = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmQ);
    ptx::prefetch_tensormap(&tmK);
    ptx::prefetch_tensormap(&tmV);
  }
  if (warp == 4) {
    ptx::tmem_alloc(tmem_slot, 256);
    ptx::tmem_relinquish_alloc_permit();
  }
  grid_dependency_wait();
  const int groups = p.hk * p.nsub;
  const int hs = static_cast<int>(blockIdx.x) % groups;
  Item it{};
  const bool live = plan_item(p.plan, p.gran, static_cast<int>(blockIdx.x) / groups, lane, &it);
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;

  const bool behind = live && it.entry == p.plan.n - 1;
  const int first = live ? (behind ? it.tile : (it.len + p.tq - 1) / p.tq - 1 - it.tile) * p.tq : 0;
  const int n = (live && !behind) ? (min(it.len, first + p.tq) + kTile - 1) / kTile : 0;  // key blocks

  // 256 x 128 registers at launch = 128 x 192 + 128 x 64
  if (warp >= 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 5 && n > 0) {
      // ---------------------------------------------------------------- loads
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(q_full, TB);
        load_tile<DT>(sQ, &tmQ, hs * p.gp, it.start + first, q_full);
      }
      uint32_t fix_phase = 0;
      bool ok = true;
      for (int j = 0; ok && j < n; ++j) {
        const uint32_t par = (j & 1) ^ 1u;
        // rows of V behind the sequence meet P = 0, which is only harmless if they are finite: they are
        // cleared before the product reads them (rows of K give columns that the mask overwrites)
        ok = ring_load<DT>(sK, &tmK, hs / p.nsub, it.start + j * kTile, kTile, k_full, s_full, par, fix, &fix_phase,
                           lane, cta_abort, p.status) &&
             ring_load<DT>(sV, &tmV, hs / p.nsub, it.start + j * kTile, min(kTile, it.len - j * kTile), v_full,
                           pv_done, par, fix, &fix_phase, lane, cta_abort, p.status);
      }
      if (!ok || *cta_abort != 0) drain_copies();
    } else if (warp == 4 && n > 0) {
      // ----------------------------------------------------------- MMA issuer
      constexpr uint32_t id_s = ptx::make_idesc(mma_fmt<T>(), false, false, 128, 128);
      constexpr uint32_t id_o = ptx::make_idesc(mma_fmt<T>(), false, true, 128, DT);
      bool ok = warp_wait(q_full, 0, cta_abort, p.status, ST_ISSUE) &&
                warp_wait(k_full, 0, cta_abort, p.status, ST_ISSUE);
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        mma_abt<DT>(tmem, sQ, sK, id_s);
        mma_commit(s_full);
      }
      for (int j = 0; ok && j < n; ++j) {
        ok = warp_wait(v_full, j & 1, cta_abort, p.status, ST_ISSUE) &&
             warp_wait(p_ready, j & 1, cta_abort, p.status, ST_ISSUE2);
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        mma_pb<DT>(tmem + 128, tmem, tmem + 32, sV, id_o, j > 0);
        mma_commit(pv_done);
        if (j + 1 < n) {
          ok = warp_wait(k_full, (j + 1) & 1, cta_abort, p.status, ST_ISSUE);
          if (!ok) break;
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tmem, sQ, sK, id_s);
          mma_commit(s_full);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ------------------------------------------------- softmax and epilogue
    const int row = warp * 32 + lane;
    const int tok = first + (row >> p.gp_shift);
    const int head = hs * p.gp + (row & (p.gp - 1));
    const int64_t token = static_cast<int64_t>(it.start) + tok;
    const bool row_ok = live && tok < it.len;
    const int64_t out_at = token * p.o.st + head * p.o.sh;
    T* out = static_cast<T*>(p.o.ptr) + out_at;
    if (behind && row_ok)  // (the gradients of these rows are zeros whatever the residual holds)
      for (int c = 0; c < p.d; c += 8) st_global_v4(out + c, make_uint4(0, 0, 0, 0));
    if (n > 0) {
      const uint32_t ts = tmem + (static_cast<uint32_t>(warp * 32) << 16), to = ts + 128;
      const int lim = min(tok, it.len - 1);     // last key this row sees
      const int safe = min(first, it.len - 1);  // last key that every row of the tile sees
      const float c = p.scale_log2;
      float m = 0.f, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        ok = warp_wait(s_full, j & 1, cta_abort, p.status, ST_MATH);
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        float s[128];
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(ts + q * 32, s + q * 32);
        tmem_wait_ld();
        if (j * kTile + kTile - 1 > safe) {
          const int last = lim - j * kTile;
#pragma unroll
          for (int e = 0; e < 128; ++e) s[e] = e <= last ? s[e] : -INFINITY;
        }
        float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
        for (int e = 4; e < 124; e += 8) {
#pragma unroll
          for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], fmaxf(s[e + q], s[e + 4 + q]));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) mx[q] = fmaxf(mx[q], s[124 + q]);
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        if (j == 0) {
          m = fmaxf(top, -1e30f);  // finite, should a whole block score -inf
        } else if (__any_sync(0xffffffffu, (top - m) * c > kLazyMax)) {
          // (the blocks before are in O: scores j were computed behind them)
          const float nm = fmaxf(m, top);
          const float alpha = ex2((m - nm) * c);
          m = nm;
          l *= alpha;
#pragma unroll 1
          for (int q = 0; q < DT / 32; ++q) {
            float o[32];
            tmem_ld32(to + q * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= alpha;
            tmem_st32(to + q * 32, o);
          }
        }
        const f32x2 c2 = pair(c, c), mc2 = pair(-m * c, -m * c);
        f32x2 sum2 = pair(0.f, 0.f);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const f32x2 x = fma2(pair(s[q * 32 + 2 * e], s[q * 32 + 2 * e + 1]), c2, mc2);
            const float a = ex2(lo_of(x)), b = ex2(hi_of(x));
            sum2 = add2(sum2, pair(a, b));
            pk[e] = pack2<T>(a, b);  // the product's operand type; the sum keeps fp32
          }
          tmem_st16(ts + q * 16, pk);
        }
        tmem_wait_st();
        ptx::tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(p_ready);
        l += lo_of(sum2) + hi_of(sum2);
      }
      ok = ok && warp_wait(pv_done, (n - 1) & 1, cta_abort, p.status, ST_MATH);
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        const float inv = 1.0f / l;
        if (row_ok && p.lse2 != nullptr) p.lse2[static_cast<int64_t>(head) * p.total + token] = m * c + log2f(l);
        if (first + p.tq <= it.len) {  // into Q's place, the residual into K's
          const uint32_t lo_tile = p.o_lo != nullptr ? sK : 0u;
#pragma unroll 1
          for (int c = 0; c < DT; c += 32) stage_cols<T>(to + c, sQ, lo_tile, row, c, inv);
          store_tile<DT>(warp == 0 && lane == 0, staged, sQ, &tmO, lo_tile, &tmL, hs * p.gp, it.start + first, lane,
                         cta_abort, p.status);
        } else {
          T* lo = p.o_lo != nullptr ? static_cast<T*>(p.o_lo) + out_at : nullptr;
#pragma unroll 1
          for (int c = 0; c < DT; c += 32) store_cols<T>(to + c, out, lo, c, p.d, inv, row_ok);
        }
      }
    }
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 4) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem, 256);
  }
}

template <typename T, int DT>
int launch_fwd(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const CUtensorMap& o,
               const CUtensorMap& l, const Params& p, int64_t batch, cudaStream_t s) {
  auto* kern = attn_fwd_kernel<T, DT>;
  static std::atomic<uint64_t> reserved{0};
  BT_CHECK_LAUNCHED(reserve_smem(kern, FwdGeo<DT>::kSmem, &reserved), "attn_fwd: shared memory");
  const int64_t grid = max_items(p.total, batch, p.tq) * p.hk * p.nsub;
  BT_CHECK_ARG(grid <= 0x7fffffffll, "attn_fwd: too many tiles (%lld)", (long long)grid);
  BT_CHECK_LAUNCHED(launch_dependent(kern, dim3(static_cast<unsigned>(grid)), dim3(kFwdThreads), FwdGeo<DT>::kSmem, s,
                                     q, k, v, o, l, p),
                    "attn_fwd");
  return BT_OK;
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<EncodeTiledFn>(ptr);
  });
  return fn;
}

}  // namespace

int check_view(const char* what, const void* p, int64_t st, int64_t sh, int heads, int64_t total) {
  BT_CHECK_ARG(p != nullptr, "%s: null pointer", what);
  BT_CHECK_ARG(aligned16(p), "%s: must be 16-byte aligned", what);
  BT_CHECK_ARG((total <= 1 || (st > 0 && st % 8 == 0)) && (heads <= 1 || (sh > 0 && sh % 8 == 0)),
               "%s: token and head strides must be positive multiples of 8 elements", what);
  return BT_OK;
}

int encode_rows(CUtensorMap* tm, const void* ptr, int dtype, int d, int heads, int64_t total, int64_t sh, int64_t st,
                int box_heads, int box_tokens, const char* what) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) {
    set_error("cuTensorMapEncodeTiled is not available from this driver");
    return BT_ERR_DRIVER;
  }
  // the stride of a dimension of one element is never used, but it has to be a valid one
  const int64_t row = (d + 7) / 8 * 8;
  if (heads <= 1) sh = row;
  if (total <= 1) st = row * heads;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(heads),
                              static_cast<cuuint64_t>(total)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(sh) * 2, static_cast<cuuint64_t>(st) * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = fn(tm, dtype == BT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                        const_cast<void*>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                        CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("%s: cuTensorMapEncodeTiled failed with CUresult %d (%d x %d x %lld, strides %lld %lld)", what,
              static_cast<int>(r), d, heads, (long long)total, (long long)sh, (long long)st);
    return BT_ERR_DRIVER;
  }
  return BT_OK;
}

int fill_params(Params* p, const char* what, const int32_t* plan, int64_t batch, int64_t total, int64_t hq, int64_t hk,
                int64_t d, float scale, int dtype) {
  BT_CHECK_ARG(dtype == BT_BF16 || dtype == BT_FP16, "%s: dtype must be bf16 or fp16 (got %d)", what, dtype);
  BT_CHECK_ARG(plan != nullptr, "%s: null plan", what);
  BT_CHECK_ARG(batch >= 0 && batch < (1 << 24) && total > 0 && total < (1ll << 30), "%s: bad batch or token count",
               what);
  BT_CHECK_ARG(hk >= 1 && hq >= hk && hq % hk == 0 && hq <= 65536,
               "%s: query heads must be a multiple of key/value heads", what);
  BT_CHECK_ARG(d >= 8 && d <= 128 && d % 8 == 0, "%s: head_dim must be a multiple of 8, at most 128 (got %lld)", what,
               (long long)d);
  // (zero would multiply the masked scores, -inf)
  BT_CHECK_ARG(scale >= 1e-30f && scale <= 1e30f, "%s: scale must be between 1e-30 and 1e30 (got %g)", what, scale);
  p->plan.words = plan;
  p->plan.n = static_cast<int>(batch) + 1;
  p->hq = static_cast<int>(hq);
  p->hk = static_cast<int>(hk);
  p->d = static_cast<int>(d);
  p->total = static_cast<int>(total);
  const int group = static_cast<int>(hq / hk);
  p->gp = 1;
  p->gp_shift = 0;
  while (p->gp < 16 && group % (2 * p->gp) == 0) {
    p->gp *= 2;
    ++p->gp_shift;
  }
  p->nsub = group / p->gp;
  p->tq = kTile / p->gp;
  p->scale = scale;
  p->scale_log2 = scale * kLog2e;
  return BT_OK;
}

}  // namespace attn
}  // namespace bt

int bt_internal_set_wait_limit_attn_fwd(unsigned long long ns) {
  return bt::ptx::set_wait_limit_ns(ns) == cudaSuccess ? 0 : -1;
}

extern "C" int64_t bt_attn_plan_words(int64_t batch) { return batch < 0 ? 0 : bt::attn::plan_words(batch); }

extern "C" int bt_attn_plan(const int32_t* cu_seqlens, int64_t batch, int64_t total, int32_t* plan, int32_t* status,
                            void* stream) {
  using namespace bt;
  BT_CHECK_ARG(batch >= 0 && batch < (1 << 24) && total >= 0 && total < (1ll << 30),
               "attn_plan: bad batch or token count");
  BT_CHECK_ARG(cu_seqlens != nullptr && plan != nullptr, "attn_plan: null pointer");
  BT_CHECK_LAUNCHED(launch_dependent(attn::attn_plan_kernel, dim3(1), dim3(attn::kPlanThreads), 0,
                                     static_cast<cudaStream_t>(stream), cu_seqlens, static_cast<int>(batch),
                                     static_cast<int>(total), plan, status),
                    "attn_plan");
  return BT_OK;
}

extern "C" int bt_attn_fwd(const void* q, const void* k, const void* v, void* out, void* out_lo, float* lse2,
                           const int32_t* plan, int64_t batch, int64_t total, int64_t hq, int64_t hk, int64_t d,
                           const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                           const int64_t* o_strides, float scale, int dtype, int32_t* status, void* stream) {
  using namespace bt;
  using namespace bt::attn;
  Params p{};
  if (int rc = fill_params(&p, "attn_fwd", plan, batch, total, hq, hk, d, scale, dtype)) return rc;
  const int nq = static_cast<int>(hq), nk = static_cast<int>(hk), nd = static_cast<int>(d);
  BT_CHECK_ARG(q_strides && k_strides && v_strides && o_strides, "attn_fwd: null strides");
  if (int rc = check_view("attn_fwd q", q, q_strides[0], q_strides[1], nq, total)) return rc;
  if (int rc = check_view("attn_fwd k", k, k_strides[0], k_strides[1], nk, total)) return rc;
  if (int rc = check_view("attn_fwd v", v, v_strides[0], v_strides[1], nk, total)) return rc;
  if (int rc = check_view("attn_fwd out", out, o_strides[0], o_strides[1], nq, total)) return rc;
  BT_CHECK_ARG(aligned16(out_lo), "attn_fwd out_lo: must be 16-byte aligned");
  p.gran = gran_index(p.tq);
  p.o_lo = out_lo;
  p.lse2 = lse2;
  p.o = View{out, o_strides[0], o_strides[1]};
  p.status = status;
  bind_context();
  CUtensorMap tq, tk, tv, to, tl;
  if (int rc = encode_rows(&tq, q, dtype, nd, nq, total, q_strides[1], q_strides[0], p.gp, p.tq, "attn_fwd q"))
    return rc;
  if (int rc = encode_rows(&tk, k, dtype, nd, nk, total, k_strides[1], k_strides[0], 1, kTile, "attn_fwd k")) return rc;
  if (int rc = encode_rows(&tv, v, dtype, nd, nk, total, v_strides[1], v_strides[0], 1, kTile, "attn_fwd v")) return rc;
  if (int rc = encode_rows(&to, out, dtype, nd, nq, total, o_strides[1], o_strides[0], p.gp, p.tq, "attn_fwd out"))
    return rc;
  tl = to;
  if (out_lo != nullptr) {
    if (int rc = encode_rows(&tl, out_lo, dtype, nd, nq, total, o_strides[1], o_strides[0], p.gp, p.tq,
                             "attn_fwd out_lo"))
      return rc;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BT_BF16)
    return d <= 64 ? launch_fwd<__nv_bfloat16, 64>(tq, tk, tv, to, tl, p, batch, s)
                   : launch_fwd<__nv_bfloat16, 128>(tq, tk, tv, to, tl, p, batch, s);
  return d <= 64 ? launch_fwd<__half, 64>(tq, tk, tv, to, tl, p, batch, s)
                 : launch_fwd<__half, 128>(tq, tk, tv, to, tl, p, batch, s);
}
