// Causal attention over packed sequences, backward.  With P = exp(scale S - lse), D_i = dO_i . O_i:
//
//   dV_j = sum_i P_ij dO_i     dS_ij = P_ij (dO_i . V_j - D_i)
//   dK_j = scale sum_i dS_ij Q_i     dQ_i = scale sum_j dS_ij K_j
//
// Two kernels, each with its sums in tensor memory from the first tile to the last and one store at
// the end: dK and dV per key tile (query rows of all heads of the group are rows of the same tiles),
// dQ per query tile.  S and dO V^T are computed by both - seven products where one kernel could do
// with five - but that one would have to add dQ tiles into memory by atomics, whose order changes
// the result; here every launch gives the same bits.
// P and dS are rounded to 16 bits, the operands' type (fp16: scaled by powers of two, see ds_scale and kPUp):
// gradients are off by 2.4e-3 of their 2-norm with bf16 and 3.0e-4 with fp16, of which the rounding of the
// results is 1.7e-3 and 2.1e-4.
// Measured, 8192 tokens in one sequence, 32 / 8 heads of 128, bf16: dK and dV 777 us, dQ 591 us, which is
// 1.41 and 1.39 PFLOP/s of the products that they execute (a library product of this length runs at 1.41:
// the chip's power limit, at 1.4 - 1.5 GHz); D = dO . O 35 us.  fp16: 808, 623 and 41 us (max|V| is read too).
// At 4096 tokens the matrix pipe is busy in 66% and 60% of the cycles, the exponentials' in 36% and 42%.
#include "attn_sm100.cuh"

namespace bt {
namespace attn {
namespace {

constexpr int kBwdThreads = 384;

// ------------------------------------------------------------------ D = dO . O
// Half a warp per (token, head) row, 16 bytes of each tensor per lane, four rows in flight.  Bound by
// memory.  O comes as its 16-bit values and what their rounding cut off: with the rounded O alone, D is
// off by dO . (that), which is as much in dQ and dK as the rounding of dS (2-norm of the error of dQ at
// bf16: 2.7e-3 instead of 2.4e-3; 1.7e-3 is the rounding of the result).
template <typename T>
constexpr bool kScaled = std::is_same<T, __half>::value;

// What fp16 wants to know of V and the sequences besides.
template <typename T>
struct BoundArgs {
  const T* v;
  int64_t v_st, v_sh;
  int hk;
  const int32_t* covered;  // tokens of sequences
  float2* out;             // one per block
};

template <typename T>
__device__ __forceinline__ float greatest(const float (&x)[8], float m) {
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fabsf(x[e]) <= 65504.f ? fmaxf(m, fabsf(x[e])) : m;
  return m;
}

template <typename T>
__global__ void __launch_bounds__(256)
attn_delta_kernel(const T* __restrict__ out, const T* __restrict__ out_lo, const T* __restrict__ dout,
                  float* __restrict__ delta, int64_t rows, int heads, int64_t total, int d, int64_t o_st, int64_t o_sh,
                  int64_t g_st, int64_t g_sh, const BoundArgs<T> bound) {
  grid_dependency_wait();
  constexpr int kRows = 4;
  const int covered = kScaled<T> ? __ldg(bound.covered) : 0;
  float max_g = 0.f, max_v = 0.f;
  const int sub = threadIdx.x & 15;
  const bool live = sub * 8 < d;
  const bool small = rows <= 0xffffffffll;  // a 64-bit division costs more than the row's arithmetic
  const int64_t step = static_cast<int64_t>(gridDim.x) * 16 * kRows;
  for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * 16 * kRows; r0 < rows; r0 += step) {
    uint4 a[kRows], b[kRows], c[kRows];
    int64_t at[kRows], tok_of[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int64_t r = r0 + i * 16 + (threadIdx.x >> 4);
      a[i] = b[i] = c[i] = make_uint4(0, 0, 0, 0);
      at[i] = -1;
      tok_of[i] = 0;
      if (r < rows) {
        const int64_t tok = small ? static_cast<uint32_t>(r) / static_cast<uint32_t>(heads) : r / heads;
        const int64_t head = r - tok * heads;
        at[i] = head * total + tok;
        tok_of[i] = tok;
        if (live) {
          a[i] = ld_stream_v4(out + tok * o_st + head * o_sh + sub * 8);
          if (out_lo != nullptr) c[i] = ld_stream_v4(out_lo + tok * o_st + head * o_sh + sub * 8);
          b[i] = ld_global_v4(dout + tok * g_st + head * g_sh + sub * 8);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      float x[8], y[8], z[8], acc = 0.f;
      Cvt<T>::unpack(a[i], x);
      Cvt<T>::unpack(b[i], y);
      Cvt<T>::unpack(c[i], z);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc = fmaf(x[e] + z[e], y[e], acc);
      if (kScaled<T> && tok_of[i] < covered) max_g = greatest<T>(y, max_g);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
      if (at[i] >= 0 && sub == 0) delta[at[i]] = acc;
    }
  }
  if constexpr (kScaled<T>) {
    const int64_t v_rows = static_cast<int64_t>(covered) * bound.hk;
    for (int64_t r0 = static_cast<int64_t>(blockIdx.x) * 16 * kRows; r0 < v_rows; r0 += step) {
      uint4 a[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int64_t r = r0 + i * 16 + (threadIdx.x >> 4);
        a[i] = make_uint4(0, 0, 0, 0);
        if (r < v_rows && live) {
          const int64_t tok = small ? static_cast<uint32_t>(r) / static_cast<uint32_t>(bound.hk) : r / bound.hk;
          a[i] = ld_global_v4(bound.v + tok * bound.v_st + (r - tok * bound.hk) * bound.v_sh + sub * 8);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        float x[8];
        Cvt<T>::unpack(a[i], x);
        max_v = greatest<T>(x, max_v);
      }
    }
    __shared__ float2 s_max[8];
    // (bits of non-negative floats are ordered as integers)
    const float g = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(max_g)));
    const float v = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(max_v)));
    if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = make_float2(g, v);
    __syncthreads();
    if (threadIdx.x == 0) {
      float2 m = s_max[0];
      for (int i = 1; i < 8; ++i) m.x = fmaxf(m.x, s_max[i].x), m.y = fmaxf(m.y, s_max[i].y);
      bound.out[blockIdx.x] = m;
    }
  }
}

// 2^k of dS, the same in every CTA; `place` has room for a float2 per warp.  About 1000 values from L2 before
// a CTA's first load: 0.4 - 0.6 us of 12 - 22 in dQ and dK/dV of 64 short sequences (fp16 alone).
template <typename T>
__device__ __forceinline__ float ds_scale(const Params& p, float2* place) {
  if constexpr (!kScaled<T>) {
    return 1.f;
  } else {
    float2 m = make_float2(0.f, 0.f);
    for (int i = threadIdx.x; i < p.n_bounds; i += kBwdThreads) {
      const float2 b = __ldg(p.bounds + i);
      m.x = fmaxf(m.x, b.x), m.y = fmaxf(m.y, b.y);
    }
    m.x = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(m.x)));
    m.y = __int_as_float(__reduce_max_sync(0xffffffffu, __float_as_int(m.y)));
    if ((threadIdx.x & 31) == 0) place[threadIdx.x >> 5] = m;
    __syncthreads();
    for (int i = 0; i < kBwdThreads / 32; ++i) m.x = fmaxf(m.x, place[i].x), m.y = fmaxf(m.y, place[i].y);
    const float most = 2.f * p.d * m.x * m.y;
    int e;
    frexpf(most, &e);
    return most > 0.f ? ldexpf(1.f, min(15 - e, 60)) : 1.f;
  }
}
// fp16: P^T, at most 1, is the operand of dV as 2^15 P^T, for the probabilities of long rows and of keys that
// are hardly seen (2^-14 is the smallest that fp16 holds at full precision).  The power goes into the
// exponent, and out of dV and of the scale of dS.
template <typename T>
constexpr float kPUp = kScaled<T> ? 15.f : 0.f;
template <typename T>
constexpr float kPDown = kScaled<T> ? 1.f / 32768.f : 1.f;
// 2^k (dP - D), D scaled before
template <typename T>
__device__ __forceinline__ f32x2 minus_d(f32x2 dp, f32x2 scale, f32x2 minus_scaled_d) {
  return kScaled<T> ? fma2(dp, scale, minus_scaled_d) : add2(dp, minus_scaled_d);
}

template <int DT>
struct BwdGeo {
  static constexpr int kTileBytes = (DT / 64) * kBoxBytes;
  static constexpr int kVecBytes = 2 * 2 * 128 * 4;  // two stages of -lse and -D of a query tile
  // K, V, three Q and two dO tiles (dK, dV), or Q, dO, three K and two V tiles (dQ); no slack to
  // align the start: the kernels check that the dynamic shared memory starts on 1024 bytes
  static constexpr int kSmem = 7 * kTileBytes + kVecBytes + 512;
};

// ----------------------------------------------------------------- dK and dV
// One CTA per (128 keys, key/value head).  Warps 0..7: one key row and half of the 128 query columns
// per thread; warp 8 issues, warp 9 loads.  Transposed scores, so that P^T and dS^T are the
// tensor-memory operands of the two sums:
//   S^T = K Q_i^T ; dP^T = V dO_i^T ; dV += P^T dO_i ; dK += dS^T Q_i
// Tensor memory is full (S^T, dP^T, dV, dK: 128 columns each), so the 16-bit P^T and dS^T replace dP^T:
// a warp writes both into the 64 columns that it has just read, P^T in the first 32.  S^T is free as
// soon as it is in registers, and S^T of the next tile is computed under this tile's dS phase; the
// exponentials of the next tile then run under dV, dK and dP^T.
//
// PAIR: clusters of two CTAs.  The first key tile of a sequence has all its query tiles to go through,
// 1.75 us each, while the rest of a short batch is long done.  Where that is more than twice the time of
// an even deal (L / TQ of the longest sequence against the sum of L (L + 128) / (256 TQ) over all, heads
// times, on all SMs) both CTAs of a cluster take half of a key tile's query tiles, and each gets one of the
// other's two sums through distributed shared memory; else they take a key tile each.  Twice, because the
// 5 us that a CTA needs besides its query tiles are paid twice.  Measured, alone / shared, us (key/value
// heads x tokens, 4 query heads each, d = 128, bf16; the even deal as a part of the longest): 8 x 1024
// (0.24) 56 / 35, 2 x 8192 (0.44) 380 / 204, 8 x 2048 (0.46) 106 / 67, a ragged batch of 8 x 4096 (0.66)
// 79 / 95, 2 x 16384 (0.87) 809 / 766, 8 x 4096 (0.89) 207 / 217, 8 x two of 2048 (0.92) 113 / 134.
template <typename T, int DT, bool PAIR>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dkv_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG, const Params p) {
  using G = BwdGeo<DT>;
  constexpr int TB = G::kTileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (!aligned_start(smem, p.status)) return;
  const uint32_t sK = ptx::smem_u32(smem), sV = sK + TB, sQ = sK + 2 * TB, sG = sK + 5 * TB;
  float* vec = reinterpret_cast<float*>(smem + 7 * TB);  // [stage][-lse | -D][128]
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + 7 * TB + G::kVecBytes);
  uint64_t* v_full = k_full + 1;
  uint64_t* q_full = v_full + 1;      // [3]
  uint64_t* q_empty = q_full + 3;     // [3]
  uint64_t* g_full = q_empty + 3;     // [2]
  uint64_t* g_empty = g_full + 2;     // [2]
  uint64_t* vec_full = g_empty + 2;   // [2]
  uint64_t* vec_empty = vec_full + 2; // [2]
  uint64_t* s_full = vec_empty + 2;
  uint64_t* s_free = s_full + 1;
  uint64_t* dp_full = s_free + 1;
  uint64_t* ds_ready = dp_full + 1;
  uint64_t* done = ds_ready + 1;
  uint64_t* fix = done + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fix + 1);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    ptx::mbar_init(k_full, 1);
    ptx::mbar_init(v_full, 1);
    for (int i = 0; i < 3; ++i) {
      ptx::mbar_init(&q_full[i], 1);
      ptx::mbar_init(&q_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&g_full[i], 1);
      ptx::mbar_init(&g_empty[i], 1);
      ptx::mbar_init(&vec_full[i], 32);
      ptx::mbar_init(&vec_empty[i], 8);
    }
    ptx::mbar_init(s_full, 1);
    ptx::mbar_init(s_free, 8);
    ptx::mbar_init(dp_full, 1);
    ptx::mbar_init(ds_ready, 8);
    ptx::mbar_init(done, 1);
    ptx::mbar_init(fix, 1);
    *cta_abort = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmQ);
    ptx::prefetch_tensormap(&tmK);
    ptx::prefetch_tensormap(&tmV);
    ptx::prefetch_tensormap(&tmG);
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish_alloc_permit();
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  const float ds_up = ds_scale<T>(p, reinterpret_cast<float2*>(smem + 7 * TB + G::kVecBytes + 256));
  const float dk_scale = kScaled<T> ? p.scale / ds_up : p.scale;
  const float up = ds_up * kPDown<T>;

  const bool shared_tiles = PAIR && p.plan.area() < p.share * static_cast<float>(p.plan.longest());
  const int unit = static_cast<int>(shared_tiles ? blockIdx.x / 2 : blockIdx.x);
  const int hk = unit % p.hk;
  Item it{};
  const bool live = plan_item(p.plan, p.gran, unit / p.hk, lane, &it);
  const bool behind = live && it.entry == p.plan.n - 1;
  const int kv0 = live ? it.tile * kTile : 0;
  const int i0 = kv0 / p.tq;                                     // first query tile that sees a key of this one
  const int per = live ? (it.len + p.tq - 1) / p.tq - i0 : 0;    // query tiles of one packed group
  const int all = (live && !behind) ? per * p.nsub : 0;
  // this CTA's query tiles are `all` of them from x0 on, n of them; with few, the first CTA takes all
  const int rank = shared_tiles ? static_cast<int>(blockIdx.x & 1) : 0;
  const bool sharing = shared_tiles && all >= 4;
  const int x0 = sharing && rank != 0 ? (all + 1) / 2 : 0;
  const int n = sharing ? (rank != 0 ? all / 2 : (all + 1) / 2) : (rank != 0 ? 0 : all);

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 9 && n > 0) {
      // ---------------------------------------------------------------- loads
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(k_full, TB);
        load_tile<DT>(sK, &tmK, hk, it.start + kv0, k_full);
        ptx::mbar_arrive_expect_tx(v_full, TB);
        load_tile<DT>(sV, &tmV, hk, it.start + kv0, v_full);
      }
      uint32_t fix_phase = 0;
      bool ok = true;
      int sub = x0 / per, i = i0 + x0 % per;
      int qs = 0;
      uint32_t q_par = 1;
      for (int x = 0; ok && x < n; ++x) {
        const int st = x & 1;
        const uint32_t par = ((x >> 1) & 1) ^ 1u;
        const int head = (hk * p.nsub + sub) * p.gp;
        const int tok0 = i * p.tq;
        const int valid = min(p.tq, it.len - tok0) << p.gp_shift;
        // rows of Q and dO behind the sequence are cleared: they meet P = dS = 0, as the rest of a
        // product they only have to be finite
        ok = ring_load<DT>(sQ + qs * TB, &tmQ, head, it.start + tok0, valid, &q_full[qs], &q_empty[qs], q_par, fix,
                           &fix_phase, lane, cta_abort, p.status) &&
             __all_sync(0xffffffffu, ptx::mbar_wait(&vec_empty[st], par, cta_abort, p.status, ST_LOAD));
        if (!ok) break;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = e * 32 + lane;
          const int token = it.start + tok0 + (r >> p.gp_shift);
          const int64_t at = static_cast<int64_t>(head + (r & (p.gp - 1))) * p.total + token;
          const bool in = r < valid;
          vec[st * 256 + r] = in ? kPUp<T> - __ldg(p.lse2 + at) : -INFINITY;  // no row: P = 0
          vec[st * 256 + 128 + r] = in ? -__ldg(p.delta + at) * up : 0.f;
        }
        ptx::mbar_arrive(&vec_full[st]);
        ok = ring_load<DT>(sG + st * TB, &tmG, head, it.start + tok0, valid, &g_full[st], &g_empty[st], par, fix,
                           &fix_phase, lane, cta_abort, p.status);
        if (++i == i0 + per) {
          i = i0;
          ++sub;
        }
        if (++qs == 3) {
          qs = 0;
          q_par ^= 1u;
        }
      }
      if (!ok || *cta_abort != 0) drain_copies();
    } else if (warp == 8 && n > 0) {
      // ----------------------------------------------------------- MMA issuer
      constexpr uint32_t id_s = ptx::make_idesc(mma_fmt<T>(), false, false, 128, 128);
      constexpr uint32_t id_o = ptx::make_idesc(mma_fmt<T>(), false, true, 128, DT);
      const uint32_t tS = tmem, tP = tmem + 128, tV = tmem + 256, tK = tmem + 256 + DT;
      bool ok = warp_wait(k_full, 0, cta_abort, p.status, ST_ISSUE) &&
                warp_wait(&q_full[0], 0, cta_abort, p.status, ST_ISSUE);
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        mma_abt<DT>(tS, sK, sQ, id_s);
        mma_commit(s_full);
        ok = warp_wait(v_full, 0, cta_abort, p.status, ST_ISSUE) &&
             warp_wait(&g_full[0], 0, cta_abort, p.status, ST_ISSUE);
      }
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        mma_abt<DT>(tP, sV, sG, id_s);
        mma_commit(dp_full);
      }
      if (ok && n > 1) {
        ok = warp_wait(&q_full[1], 0, cta_abort, p.status, ST_ISSUE) &&
             warp_wait(s_free, 0, cta_abort, p.status, ST_ISSUE2);
        if (ok) {
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tS, sK, sQ + TB, id_s);
          mma_commit(s_full);
        }
      }
      int qs = 0, q2 = 2;  // Q stages of tiles x and x + 2
      uint32_t q2_par = 0;
      for (int x = 0; ok && x < n; ++x) {
        const int st = x & 1, nst = st ^ 1;
        ok = warp_wait(ds_ready, x & 1, cta_abort, p.status, ST_ISSUE2);
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        mma_pb<DT>(tV, tP, tP + 64, sG + st * TB, id_o, x > 0);
        mma_commit(&g_empty[st]);
        mma_pb<DT>(tK, tP + 32, tP + 96, sQ + qs * TB, id_o, x > 0);
        mma_commit(&q_empty[qs]);
        qs = qs == 2 ? 0 : qs + 1;
        if (x + 1 < n) {
          ok = warp_wait(&g_full[nst], ((x + 1) >> 1) & 1, cta_abort, p.status, ST_ISSUE);
          if (!ok) break;
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tP, sV, sG + nst * TB, id_s);
          mma_commit(dp_full);
        }
        if (x + 2 < n) {
          ok = warp_wait(&q_full[q2], q2_par, cta_abort, p.status, ST_ISSUE) &&
               warp_wait(s_free, (x + 1) & 1, cta_abort, p.status, ST_ISSUE2);
          if (!ok) break;
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tS, sK, sQ + q2 * TB, id_s);
          mma_commit(s_full);
          if (++q2 == 3) {
            q2 = 0;
            q2_par ^= 1u;
          }
        }
      }
      if (ok) mma_commit(done);
    }
    if (PAIR && sharing) {
      __syncwarp();
      ptx::cluster_sync_all();
      ptx::cluster_sync_all();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // --------------------------------------------------------- P^T, dS^T, stores
    const int half = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int kv = kv0 + row;
    if (behind && rank == 0 && kv < it.len) {
      const int64_t token = static_cast<int64_t>(it.start) + kv;
      T* dk = static_cast<T*>(p.dk.ptr) + token * p.dk.st + hk * p.dk.sh;
      T* dv = static_cast<T*>(p.dv.ptr) + token * p.dv.st + hk * p.dv.sh;
      for (int c = half * 8; c < p.d; c += 16) {
        st_global_v4(dk + c, make_uint4(0, 0, 0, 0));
        st_global_v4(dv + c, make_uint4(0, 0, 0, 0));
      }
    }
    if (n > 0) {
      const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t ts = tmem + lane_base + half * 64, tp = ts + 128;
      const f32x2 c2 = pair(p.scale_log2, p.scale_log2), up2 = pair(up, up);
      bool ok = true;
      int i = i0 + x0 % per;
      for (int x = 0; x < n; ++x) {
        const int st = x & 1;
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&vec_full[st], (x >> 1) & 1, cta_abort, p.status, ST_MATH) &&
                                         ptx::mbar_wait(s_full, x & 1, cta_abort, p.status, ST_MATH));
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        const float4* nl = reinterpret_cast<const float4*>(vec + st * 256 + half * 64);
        const float4* dl = nl + 32;
        float s[64];
        tmem_ld32(ts, s);
        tmem_ld32(ts + 32, s + 32);
        tmem_wait_ld();
        ptx::tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(s_free);
        const int tok0 = i * p.tq;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float4 l4 = nl[e];
          const f32x2 a = fma2(pair(s[4 * e], s[4 * e + 1]), c2, pair(l4.x, l4.y));
          const f32x2 b = fma2(pair(s[4 * e + 2], s[4 * e + 3]), c2, pair(l4.z, l4.w));
          s[4 * e] = ex2(lo_of(a));
          s[4 * e + 1] = ex2(hi_of(a));
          s[4 * e + 2] = ex2(lo_of(b));
          s[4 * e + 3] = ex2(hi_of(b));
        }
        if (tok0 < kv0 + kTile - 1) {  // the diagonal: query rows before this key
          const int lo = (max(kv - tok0, 0) << p.gp_shift) - half * 64;
#pragma unroll
          for (int e = 0; e < 64; ++e) s[e] = e >= lo ? s[e] : 0.f;
        }
        uint32_t pp[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) pp[e] = pack2<T>(s[2 * e], s[2 * e + 1]);

        ok = __all_sync(0xffffffffu, ptx::mbar_wait(dp_full, x & 1, cta_abort, p.status, ST_MATH));
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        float dp[64];
        tmem_ld32(tp, dp);
        tmem_ld32(tp + 32, dp + 32);
        tmem_wait_ld();
        tmem_st16(tp, pp);
        tmem_st16(tp + 16, pp + 16);
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 d4 = dl[g * 8 + e];
            const int b = g * 32 + 4 * e;
            const f32x2 u = mul2(pair(s[b], s[b + 1]), minus_d<T>(pair(dp[b], dp[b + 1]), up2, pair(d4.x, d4.y)));
            const f32x2 v =
                mul2(pair(s[b + 2], s[b + 3]), minus_d<T>(pair(dp[b + 2], dp[b + 3]), up2, pair(d4.z, d4.w)));
            pk[2 * e] = pack2<T>(lo_of(u), hi_of(u));
            pk[2 * e + 1] = pack2<T>(lo_of(v), hi_of(v));
          }
          tmem_st16(tp + 32 + g * 16, pk);
        }
        tmem_wait_st();
        ptx::tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          ptx::mbar_arrive(ds_ready);
          ptx::mbar_arrive(&vec_empty[st]);
        }
        if (++i == i0 + per) i = i0;
      }
      if (ok) ok = __all_sync(0xffffffffu, ptx::mbar_wait(done, 0, cta_abort, p.status, ST_MATH));
      if (ok) ptx::tcgen05_fence_after_sync();
      const bool row_ok = kv < it.len;
      const int64_t token = static_cast<int64_t>(it.start) + kv;
      if (PAIR && sharing) {
        // the first CTA of the two ends with dV, the second with dK; whatever goes wrong in one of them, both
        // come through both barriers
        const uint32_t mine = tmem + lane_base + 256 + (rank != 0 ? DT : 0);
        const uint32_t theirs = tmem + lane_base + 256 + (rank != 0 ? 0 : DT);
        const View& view = rank != 0 ? p.dk : p.dv;
        T* dst = static_cast<T*>(view.ptr) + token * view.st + hk * view.sh;
        __syncwarp();
        ptx::cluster_sync_all();  // the products of both are done: the tiles of Q may be overwritten
        if (ok)
#pragma unroll 1
          for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32)
            send_cols(theirs + c, sQ + (c / 4 * 128 + row) * 16, static_cast<uint32_t>(rank ^ 1));
        __syncwarp();
        ptx::cluster_sync_all();
        if (ok)
#pragma unroll 1
          for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32)
            store_sum_cols<T>(mine + c, sQ + (c / 4 * 128 + row) * 16, dst, c, p.d,
                              rank != 0 ? dk_scale : kPDown<T>, row_ok);
      } else if (ok) {
        T* dk = static_cast<T*>(p.dk.ptr) + token * p.dk.st + hk * p.dk.sh;
        T* dv = static_cast<T*>(p.dv.ptr) + token * p.dv.st + hk * p.dv.sh;
        // (one store per tile and output here: a staged tile store measured 1% slower)
#pragma unroll 1
        for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32) {
          store_cols<T>(tmem + lane_base + 256 + c, dv, nullptr, c, p.d, kPDown<T>, row_ok);
          store_cols<T>(tmem + lane_base + 256 + DT + c, dk, nullptr, c, p.d, dk_scale, row_ok);
        }
      }
    }
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------ dQ
// One CTA per (query tile of 128 packed rows, key/value head).  Warps 0..7: one query row and half of
// the 128 key columns per thread.  S is double-buffered in tensor memory (its buffer then holds the
// 16-bit dS) and dP is free once it is in registers, so S_{j+1} and dP_{j+1} are ready when the math
// warps are done with tile j:
//   S = Q K_j^T ; dP = dO V_j^T ; dS = P (dP - D) ; dQ += dS K_j
template <typename T, int DT>
__global__ void __launch_bounds__(kBwdThreads, 1)
attn_dq_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
               const __grid_constant__ CUtensorMap tmV, const __grid_constant__ CUtensorMap tmG,
               const __grid_constant__ CUtensorMap tmD, const Params p) {
  using G = BwdGeo<DT>;
  constexpr int TB = G::kTileBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  if (!aligned_start(smem, p.status)) return;
  const uint32_t sQ = ptx::smem_u32(smem), sG = sQ + TB, sK = sQ + 2 * TB, sV = sQ + 5 * TB;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + 7 * TB);
  uint64_t* g_full = q_full + 1;
  uint64_t* k_full = g_full + 1;   // [3]
  uint64_t* k_empty = k_full + 3;  // [3]
  uint64_t* v_full = k_empty + 3;  // [2]
  uint64_t* v_empty = v_full + 2;  // [2]
  uint64_t* s_full = v_empty + 2;  // [2]
  uint64_t* dp_full = s_full + 2;
  uint64_t* dp_free = dp_full + 1;
  uint64_t* ds_ready = dp_free + 1;
  uint64_t* done = ds_ready + 1;
  uint64_t* staged = done + 1;
  uint64_t* fix = staged + 1;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fix + 1);
  volatile int* cta_abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    ptx::mbar_init(q_full, 1);
    ptx::mbar_init(g_full, 1);
    for (int i = 0; i < 3; ++i) {
      ptx::mbar_init(&k_full[i], 1);
      ptx::mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      ptx::mbar_init(&v_full[i], 1);
      ptx::mbar_init(&v_empty[i], 1);
      ptx::mbar_init(&s_full[i], 1);
    }
    ptx::mbar_init(dp_full, 1);
    ptx::mbar_init(dp_free, 8);
    ptx::mbar_init(ds_ready, 8);
    ptx::mbar_init(done, 1);
    ptx::mbar_init(staged, 8);
    ptx::mbar_init(fix, 1);
    *cta_abort = 0;
    ptx::fence_mbar_init();
    ptx::prefetch_tensormap(&tmQ);
    ptx::prefetch_tensormap(&tmK);
    ptx::prefetch_tensormap(&tmV);
    ptx::prefetch_tensormap(&tmG);
  }
  if (warp == 8) {
    ptx::tmem_alloc(tmem_slot, 512);
    ptx::tmem_relinquish_alloc_permit();
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  ptx::tcgen05_fence_after_sync();
  const uint32_t tmem = *tmem_slot;
  grid_dependency_wait();

  const float up = ds_scale<T>(p, reinterpret_cast<float2*>(smem + 7 * TB + G::kVecBytes + 256));

  const int groups = p.hk * p.nsub;
  const int hs = static_cast<int>(blockIdx.x) % groups;
  Item it{};
  const bool live = plan_item(p.plan, p.gran, static_cast<int>(blockIdx.x) / groups, lane, &it);
  const bool behind = live && it.entry == p.plan.n - 1;
  const int first = live ? (behind ? it.tile : (it.len + p.tq - 1) / p.tq - 1 - it.tile) * p.tq : 0;
  const int n = (live && !behind) ? (min(it.len, first + p.tq) + kTile - 1) / kTile : 0;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 9 && n > 0) {
      // ---------------------------------------------------------------- loads
      if (lane == 0) {
        ptx::mbar_arrive_expect_tx(q_full, TB);
        load_tile<DT>(sQ, &tmQ, hs * p.gp, it.start + first, q_full);
      }
      uint32_t fix_phase = 0;
      bool ok = true;
      int ks = 0;
      uint32_t k_par = 1;
      for (int j = 0; ok && j < n; ++j) {
        const int st = j & 1;
        const uint32_t par = ((j >> 1) & 1) ^ 1u;
        // K rows behind the sequence meet dS = 0 and have to be finite; V's only give masked columns
        ok = ring_load<DT>(sK + ks * TB, &tmK, hs / p.nsub, it.start + j * kTile, min(kTile, it.len - j * kTile),
                           &k_full[ks], &k_empty[ks], k_par, fix, &fix_phase, lane, cta_abort, p.status);
        if (ok && j == 0 && lane == 0) {  // behind what the first product needs
          ptx::mbar_arrive_expect_tx(g_full, TB);
          load_tile<DT>(sG, &tmG, hs * p.gp, it.start + first, g_full);
        }
        ok = ok &&
             ring_load<DT>(sV + st * TB, &tmV, hs / p.nsub, it.start + j * kTile, kTile, &v_full[st], &v_empty[st],
                           par, fix, &fix_phase, lane, cta_abort, p.status);
        if (++ks == 3) {
          ks = 0;
          k_par ^= 1u;
        }
      }
      if (!ok || *cta_abort != 0) drain_copies();
    } else if (warp == 8 && n > 0) {
      // ----------------------------------------------------------- MMA issuer
      constexpr uint32_t id_s = ptx::make_idesc(mma_fmt<T>(), false, false, 128, 128);
      constexpr uint32_t id_o = ptx::make_idesc(mma_fmt<T>(), false, true, 128, DT);
      const uint32_t tP = tmem + 256, tQ = tmem + 384;
      bool ok = warp_wait(q_full, 0, cta_abort, p.status, ST_ISSUE) &&
                warp_wait(&k_full[0], 0, cta_abort, p.status, ST_ISSUE);
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        mma_abt<DT>(tmem, sQ, sK, id_s);
        mma_commit(&s_full[0]);
        ok = warp_wait(g_full, 0, cta_abort, p.status, ST_ISSUE) &&
             warp_wait(&v_full[0], 0, cta_abort, p.status, ST_ISSUE);
      }
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        mma_abt<DT>(tP, sG, sV, id_s);
        mma_commit(dp_full);
        mma_commit(&v_empty[0]);
      }
      if (ok && n > 1) {
        ok = warp_wait(&k_full[1], 0, cta_abort, p.status, ST_ISSUE);
        if (ok) {
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tmem + 128, sQ, sK + TB, id_s);
          mma_commit(&s_full[1]);
        }
      }
      int ks = 0, k2 = 2;  // K stages of tiles j and j + 2
      uint32_t k2_par = 0;
      for (int j = 0; ok && j < n; ++j) {
        const int st = j & 1, nst = st ^ 1;
        if (j + 1 < n) {  // dP of the next tile as soon as this one's is in registers
          ok = warp_wait(&v_full[nst], ((j + 1) >> 1) & 1, cta_abort, p.status, ST_ISSUE) &&
               warp_wait(dp_free, j & 1, cta_abort, p.status, ST_ISSUE2);
          if (!ok) break;
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tP, sG, sV + nst * TB, id_s);
          mma_commit(dp_full);
          mma_commit(&v_empty[nst]);
        }
        ok = warp_wait(ds_ready, j & 1, cta_abort, p.status, ST_ISSUE2);
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        mma_pb<DT>(tQ, tmem + st * 128, tmem + st * 128 + 64, sK + ks * TB, id_o, j > 0);
        mma_commit(&k_empty[ks]);
        ks = ks == 2 ? 0 : ks + 1;
        if (j + 2 < n) {
          ok = warp_wait(&k_full[k2], k2_par, cta_abort, p.status, ST_ISSUE);
          if (!ok) break;
          ptx::tcgen05_fence_after_sync();
          mma_abt<DT>(tmem + st * 128, sQ, sK + k2 * TB, id_s);
          mma_commit(&s_full[st]);
          if (++k2 == 3) {
            k2 = 0;
            k2_par ^= 1u;
          }
        }
      }
      if (ok) mma_commit(done);
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ---------------------------------------------------------------- dS, store
    const int half = warp >> 2;
    const int row = (warp & 3) * 32 + lane;
    const int tok = first + (row >> p.gp_shift);
    const int head = hs * p.gp + (row & (p.gp - 1));
    const int64_t token = static_cast<int64_t>(it.start) + tok;
    const bool row_ok = live && tok < it.len;
    T* dq = static_cast<T*>(p.dq.ptr) + token * p.dq.st + head * p.dq.sh;
    if (behind && row_ok)
      for (int c = half * 8; c < p.d; c += 16) st_global_v4(dq + c, make_uint4(0, 0, 0, 0));
    if (n > 0) {
      const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
      const uint32_t ts0 = tmem + lane_base + half * 64, tp = ts0 + 256;
      const int64_t at = static_cast<int64_t>(head) * p.total + token;
      const float nl = row_ok ? -p.lse2[at] : -INFINITY;
      const float dl = row_ok ? -p.delta[at] * up : 0.f;
      const f32x2 c2 = pair(p.scale_log2, p.scale_log2), nl2 = pair(nl, nl), dl2 = pair(dl, dl),
                  up2 = pair(up, up);
      const int lim = min(tok, it.len - 1);
      const int safe = min(first, it.len - 1);
      bool ok = true;
      for (int j = 0; j < n; ++j) {
        const uint32_t ts = ts0 + (j & 1) * 128;
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(&s_full[j & 1], (j >> 1) & 1, cta_abort, p.status, ST_MATH));
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        float s[64];
        tmem_ld32(ts, s);
        tmem_ld32(ts + 32, s + 32);
        tmem_wait_ld();
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const f32x2 a = fma2(pair(s[2 * e], s[2 * e + 1]), c2, nl2);
          s[2 * e] = ex2(lo_of(a));
          s[2 * e + 1] = ex2(hi_of(a));
        }
        ok = __all_sync(0xffffffffu, ptx::mbar_wait(dp_full, j & 1, cta_abort, p.status, ST_MATH));
        if (!ok) break;
        ptx::tcgen05_fence_after_sync();
        float dp[64];
        tmem_ld32(tp, dp);
        tmem_ld32(tp + 32, dp + 32);
        tmem_wait_ld();
        ptx::tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(dp_free);
#pragma unroll
        for (int e = 0; e < 32; ++e) {
          const f32x2 u = mul2(pair(s[2 * e], s[2 * e + 1]), minus_d<T>(pair(dp[2 * e], dp[2 * e + 1]), up2, dl2));
          s[2 * e] = lo_of(u);
          s[2 * e + 1] = hi_of(u);
        }
        if (j * kTile + kTile - 1 > safe) {
          const int last = lim - j * kTile - half * 64;
#pragma unroll
          for (int e = 0; e < 64; ++e) s[e] = e <= last ? s[e] : 0.f;
        }
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) pk[e] = pack2<T>(s[g * 32 + 2 * e], s[g * 32 + 2 * e + 1]);
          tmem_st16(ts + g * 16, pk);
        }
        tmem_wait_st();
        ptx::tcgen05_fence_before_sync();
        __syncwarp();
        if (lane == 0) ptx::mbar_arrive(ds_ready);
      }
      if (ok) ok = __all_sync(0xffffffffu, ptx::mbar_wait(done, 0, cta_abort, p.status, ST_MATH));
      if (ok) {
        ptx::tcgen05_fence_after_sync();
        const uint32_t ta = tmem + lane_base + 384;
        const float dq_scale = kScaled<T> ? p.scale / up : p.scale;  // (only here: 1% of the time before the loop)
        if (first + p.tq <= it.len) {  // into Q's place
#pragma unroll 1
          for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32)
            stage_cols<T>(ta + c, sQ, 0, row, c, dq_scale);
          store_tile<DT>(warp == 0 && lane == 0, staged, sQ, &tmD, 0, &tmD, hs * p.gp, it.start + first, lane,
                         cta_abort, p.status);
        } else {
#pragma unroll 1
          for (int c = half * (DT / 2); c < (half + 1) * (DT / 2); c += 32)
            store_cols<T>(ta + c, dq, nullptr, c, p.d, dq_scale, row_ok);
        }
      }
    }
  }
  ptx::tcgen05_fence_before_sync();
  __syncthreads();
  if (warp == 8) {
    ptx::tcgen05_fence_after_sync();
    ptx::tmem_dealloc(tmem, 512);
  }
}

struct Maps {
  CUtensorMap q, k, v, g, dq;
};

// Key tiles are shared where the even deal, area * hk / (2 kTile * SMs), is below half of the longest
// sequence.  With sequences of one length that takes a total below this bound, which the host can see.
float share_bound(int hk) { return kTile * static_cast<float>(sm_count()) / static_cast<float>(hk); }

template <typename K, typename... A>
int launch_bwd(K* kern, int smem, std::atomic<uint64_t>* reserved, int64_t grid, int cluster, const char* what,
               cudaStream_t s, const A&... args) {
  BT_CHECK_LAUNCHED(reserve_smem(kern, smem, reserved), what);
  BT_CHECK_ARG(grid <= 0x7fffffffll, "%s: too many tiles (%lld)", what, (long long)grid);
  BT_CHECK_LAUNCHED(launch_dependent_clusters(kern, dim3(static_cast<unsigned>(grid)), dim3(kBwdThreads), smem, cluster,
                                              s, args...),
                    what);
  return BT_OK;
}

template <typename T, int DT>
int run_bwd(const Maps& m, Params p, int64_t batch, cudaStream_t s) {
  static std::atomic<uint64_t> reserved[3];
  if (p.dk.ptr != nullptr) {
    p.gran = gran_index(kTile);
    p.share = share_bound(p.hk);
    const int64_t items = max_items(p.total, batch, kTile) * p.hk;
    const int rc = static_cast<float>(p.total) < p.share
                       ? launch_bwd(attn_dkv_kernel<T, DT, true>, BwdGeo<DT>::kSmem, &reserved[2], 2 * items, 2,
                                    "attn_bwd dk, dv", s, m.q, m.k, m.v, m.g, p)
                       : launch_bwd(attn_dkv_kernel<T, DT, false>, BwdGeo<DT>::kSmem, &reserved[0], items, 1,
                                    "attn_bwd dk, dv", s, m.q, m.k, m.v, m.g, p);
    if (rc) return rc;
  }
  if (p.dq.ptr != nullptr) {
    p.gran = gran_index(p.tq);
    if (int rc = launch_bwd(attn_dq_kernel<T, DT>, BwdGeo<DT>::kSmem, &reserved[1],
                            max_items(p.total, batch, p.tq) * p.hk * p.nsub, 1, "attn_bwd dq", s, m.q, m.k, m.v, m.g,
                            m.dq, p))
      return rc;
  }
  return BT_OK;
}

template <typename T>
int run_delta(const void* out, const void* out_lo, const void* dout, const void* v, Params* p, int64_t total, int64_t hq,
              int64_t d, const int64_t* os, const int64_t* gs, const int64_t* vs, cudaStream_t s) {
  const int64_t rows = total * hq;
  const int64_t want = ceil_div(rows, 64), sms = static_cast<int64_t>(sm_count()) * 8;
  const int64_t cap = sms < kMaxBounds ? sms : kMaxBounds;
  const unsigned grid = static_cast<unsigned>(want < cap ? want : cap);
  float* delta = p->delta;
  BoundArgs<T> bound{static_cast<const T*>(v), vs[0], vs[1], p->hk, p->plan.words + p->plan.n - 1, nullptr};
  if (kScaled<T>) {  // behind D
    bound.out = reinterpret_cast<float2*>(delta + (rows + 1) / 2 * 2);
    p->bounds = bound.out;
    p->n_bounds = static_cast<int>(grid);
  }
  BT_CHECK_LAUNCHED(launch_dependent(attn_delta_kernel<T>, dim3(grid),
                                     dim3(256), 0, s, static_cast<const T*>(out), static_cast<const T*>(out_lo),
                                     static_cast<const T*>(dout), delta, rows, static_cast<int>(hq), total,
                                     static_cast<int>(d), os[0], os[1], gs[0], gs[1], bound),
                    "attn_bwd delta");
  return BT_OK;
}

}  // namespace
}  // namespace attn
}  // namespace bt

int bt_internal_set_wait_limit_attn_bwd(unsigned long long ns) {
  return bt::ptx::set_wait_limit_ns(ns) == cudaSuccess ? 0 : -1;
}

extern "C" int64_t bt_attn_delta_floats(int64_t total, int64_t hq, int dtype) {
  if (total < 0 || hq < 0) return 0;
  return dtype == BT_FP16 ? (total * hq + 1) / 2 * 2 + 2 * bt::attn::kMaxBounds : total * hq;
}

extern "C" int bt_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out,
                           const void* out_lo, const float* lse2, float* delta, void* dq, void* dk, void* dv,
                           const int32_t* plan, int64_t batch, int64_t total, int64_t hq, int64_t hk, int64_t d,
                           const int64_t* g_strides, const int64_t* q_strides, const int64_t* k_strides,
                           const int64_t* v_strides, const int64_t* o_strides, const int64_t* dq_strides,
                           const int64_t* dk_strides, const int64_t* dv_strides, float scale, int dtype,
                           int32_t* status, void* stream) {
  using namespace bt;
  using namespace bt::attn;
  Params p{};
  if (int rc = fill_params(&p, "attn_bwd", plan, batch, total, hq, hk, d, scale, dtype)) return rc;
  const int nq = static_cast<int>(hq), nk = static_cast<int>(hk), nd = static_cast<int>(d);
  BT_CHECK_ARG(lse2 != nullptr && delta != nullptr, "attn_bwd: null pointer");
  BT_CHECK_ARG(aligned16(out_lo), "attn_bwd out_lo: must be 16-byte aligned");
  BT_CHECK_ARG(reinterpret_cast<uintptr_t>(delta) % 8 == 0, "attn_bwd delta: must be 8-byte aligned");
  BT_CHECK_ARG((dk == nullptr) == (dv == nullptr), "attn_bwd: dk and dv are computed together");
  BT_CHECK_ARG(g_strides && q_strides && k_strides && v_strides && o_strides && (dq == nullptr || dq_strides) &&
                   (dk == nullptr || (dk_strides && dv_strides)),
               "attn_bwd: null strides");
  if (int rc = check_view("attn_bwd dout", dout, g_strides[0], g_strides[1], nq, total)) return rc;
  if (int rc = check_view("attn_bwd q", q, q_strides[0], q_strides[1], nq, total)) return rc;
  if (int rc = check_view("attn_bwd k", k, k_strides[0], k_strides[1], nk, total)) return rc;
  if (int rc = check_view("attn_bwd v", v, v_strides[0], v_strides[1], nk, total)) return rc;
  if (int rc = check_view("attn_bwd out", out, o_strides[0], o_strides[1], nq, total)) return rc;
  if (dq != nullptr) {
    if (int rc = check_view("attn_bwd dq", dq, dq_strides[0], dq_strides[1], nq, total)) return rc;
    p.dq = View{dq, dq_strides[0], dq_strides[1]};
  }
  if (dk != nullptr) {
    if (int rc = check_view("attn_bwd dk", dk, dk_strides[0], dk_strides[1], nk, total)) return rc;
    if (int rc = check_view("attn_bwd dv", dv, dv_strides[0], dv_strides[1], nk, total)) return rc;
    p.dk = View{dk, dk_strides[0], dk_strides[1]};
    p.dv = View{dv, dv_strides[0], dv_strides[1]};
  }
  p.lse2 = const_cast<float*>(lse2);
  p.delta = delta;
  p.status = status;
  bind_context();
  Maps m{};
  auto rows = [&](CUtensorMap* tm, const void* ptr, const int64_t* strides, bool query, const char* what) {
    if (ptr == nullptr) return BT_OK;
    return encode_rows(tm, ptr, dtype, nd, query ? nq : nk, total, strides[1], strides[0], query ? p.gp : 1,
                       query ? p.tq : kTile, what);
  };
  if (int rc = rows(&m.q, q, q_strides, true, "attn_bwd q")) return rc;
  if (int rc = rows(&m.k, k, k_strides, false, "attn_bwd k")) return rc;
  if (int rc = rows(&m.v, v, v_strides, false, "attn_bwd v")) return rc;
  if (int rc = rows(&m.g, dout, g_strides, true, "attn_bwd dout")) return rc;
  if (int rc = rows(&m.dq, dq, dq_strides, true, "attn_bwd dq")) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == BT_BF16) {
    if (int rc = run_delta<__nv_bfloat16>(out, out_lo, dout, v, &p, total, hq, d, o_strides, g_strides, v_strides, s))
      return rc;
    return d <= 64 ? run_bwd<__nv_bfloat16, 64>(m, p, batch, s) : run_bwd<__nv_bfloat16, 128>(m, p, batch, s);
  }
  if (int rc = run_delta<__half>(out, out_lo, dout, v, &p, total, hq, d, o_strides, g_strides, v_strides, s)) return rc;
  return d <= 64 ? run_bwd<__half, 64>(m, p, batch, s) : run_bwd<__half, 128>(m, p, batch, s);
}
