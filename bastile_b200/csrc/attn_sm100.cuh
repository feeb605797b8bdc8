// Shared pieces of the packed-attention kernels: the sequence plan, 3-D tile loads of head-packed
// rows, MMAs whose A operand lies in tensor memory, and the shared-memory layout of the tiles.
//
// Row packing.  With grouped heads, GP (the largest power of two that divides Hq / Hk, at most 16)
// query heads of one key/value head share a tile: row r of a 128-row query tile is token r / GP, head
// r % GP of the group.  A tile then spans TQ = 128 / GP tokens, all of its rows use the same K and V
// tiles, and sums over query rows in the backward run over the heads of the group by themselves.
//
// Every operand tile is 128 rows of DT (64 or 128) 16-bit elements, stored as DT / 64 boxes of
// 128 rows x 128 bytes with the 128-byte TMA swizzle.  A head_dim below DT is zero-filled by TMA.
#pragma once

#include <type_traits>

#include "bt_common.cuh"
#include "sm100_ptx.cuh"

namespace bt {
namespace attn {

constexpr int kTile = 128;          // rows of every operand tile
constexpr int kBoxBytes = 128 * 128;  // 128 rows x 64 16-bit elements
constexpr float kLog2e = 1.4426950408889634f;

enum : int { ST_LOAD = 1, ST_ISSUE = 2, ST_ISSUE2 = 4, ST_MATH = 8 };

// ------------------------------------------------------------------ the plan
// int32 words written once per batch by bt_attn_plan: start[n], len[n] of the n = batch + 1 entries
// (the sequences, longest first when there are at most kPlanSort of them, then the rows behind the
// last sequence), then for each tile height gran_of(g) the n + 1 running tile counts, then the sum over
// sequences of len (len + kTile) (fp32) - twice the tokens that a step through all tiles covers, times
// kTile - and the greatest length.
constexpr int kGrans = 5;
constexpr int kPlanSort = 1024;
__host__ __device__ constexpr int gran_of(int g) { return 8 << g; }
__host__ __device__ inline int gran_index(int tokens) {
  int g = 0;
  while (gran_of(g) < tokens) ++g;
  return g;
}
inline int64_t plan_words(int64_t batch) { return (batch + 1) * 2 + kGrans * (batch + 2) + 2; }

struct Plan {
  const int32_t* words;
  int n;  // entries
  __device__ __forceinline__ float area() const {
    return __int_as_float(__ldg(words + 2 * n + kGrans * (n + 1)));
  }
  __device__ __forceinline__ int longest() const { return __ldg(words + 2 * n + kGrans * (n + 1) + 1); }
};
struct Item {
  int start, len, tile, entry;  // entry == n - 1: rows behind the last sequence
};

// The item-th tile of height gran_of(g) (one warp; all lanes get the answer); false: no such tile.
// Every CTA waits for this before its first load, so the reads of a round do not wait for one another:
// up to 32 entries take one round, up to 1024 two.
__device__ __forceinline__ bool plan_item(const Plan& p, int g, int item, int lane, Item* it) {
  const int32_t* pre = p.words + 2 * p.n + g * (p.n + 1);
  const int total = __ldg(pre + p.n);
  int lo = 0, hi = p.n;
  while (hi - lo > 32) {  // invariant: pre[lo] <= item < pre[hi]; 32 probes a round
    const int step = (hi - lo + 31) / 32;
    const int at = lo + (lane + 1) * step;
    const bool le = at < hi && __ldg(pre + at) <= item;
    const int c = __popc(__ballot_sync(0xffffffffu, le));
    const int base = lo;
    lo = base + c * step;
    hi = min(base + (c + 1) * step, hi);
  }
  const int at = min(lo + lane, p.n - 1);
  const int first = __ldg(pre + at), start = __ldg(p.words + at), len = __ldg(p.words + p.n + at);
  if (item >= total) return false;
  const int src = __popc(__ballot_sync(0xffffffffu, lo + lane < hi && first <= item)) - 1;
  it->entry = lo + src;
  it->start = __shfl_sync(0xffffffffu, start, src);
  it->len = __shfl_sync(0xffffffffu, len, src);
  it->tile = item - __shfl_sync(0xffffffffu, first, src);
  return true;
}

// Grid bound for tiles of `tokens`: every entry rounds up by less than one tile.
inline int64_t max_items(int64_t total, int64_t batch, int64_t tokens) {
  return (total + (batch + 1) * (tokens - 1)) / tokens;
}

// ----------------------------------------------------------------- PTX pieces
__device__ __forceinline__ void tma_load_3d(uint32_t smem_dst, const CUtensorMap* tm, int x, int y, int z,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(tm)), "r"(x), "r"(y), "r"(z), "r"(ptx::smem_u32(bar))
      : "memory");
}
// Tile store, the way back: one box of a staged tile (rows / columns outside the tensor are clipped).
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* tm, uint32_t smem_src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
                   reinterpret_cast<uint64_t>(tm)),
               "r"(x), "r"(y), "r"(z), "r"(smem_src)
               : "memory");
}
// One operand tile: DT / 64 boxes.
template <int DT>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* tm, int head, int token, uint64_t* bar) {
#pragma unroll
  for (int j = 0; j < DT / 64; ++j) tma_load_3d(dst + j * kBoxBytes, tm, j * 64, head, token, bar);
}

// The MMA warp runs these with all lanes converged and one lane elected inside the instruction
// sequence: addresses, descriptors and predicates then stay in uniform registers, where tcgen05.mma
// takes them from.  Issued from a one-lane branch each operand is moved there first, about 80 cycles an
// MMA beside the math warps - more than the 64 that the MMA itself takes.
__device__ __forceinline__ void mma_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// A: 16-bit in tensor memory, 128 lanes, two K elements per 32-bit column.
__device__ __forceinline__ void mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@leader tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` once every MMA issued so far by the elected lane is done.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred leader;\n\t"
      "elect.sync _|leader, 0xffffffff;\n\t"
      "@leader tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(
          ptx::smem_u32(bar))
      : "memory");
}
// A wait of a whole warp: all lanes leave with the same answer.
static __device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* cta_abort,
                                                 int32_t* status, int code) {
  return __all_sync(0xffffffffu, ptx::mbar_wait(bar, parity, cta_abort, status, code));
}
// 32 columns of this thread's lane; the registers are valid after tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]),
      "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
      "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// ------------------------------------------------------- MMAs over whole tiles
// Constant halves of the shared-memory descriptors (tiles above).
constexpr uint64_t kDescK = ptx::make_smem_desc_hi(true, 0);                // rows = M/N, K along the row
constexpr uint64_t kDescMN = ptx::make_smem_desc_hi(false, kBoxBytes);      // rows = K, M/N along the row

// D[128 x 128] = A[128 x DT] B[128 x DT]^T, both from shared memory, K-major.
template <int DT>
__device__ __forceinline__ void mma_abt(uint32_t d, uint32_t a_smem, uint32_t b_smem, uint32_t idesc) {
  const uint64_t a = ptx::smem_desc(kDescK, a_smem), b = ptx::smem_desc(kDescK, b_smem);
#pragma unroll
  for (int k = 0; k < DT / 16; ++k) {
    const uint64_t off = static_cast<uint64_t>(((k / 4) * kBoxBytes + (k % 4) * 32) >> 4);
    mma_ss(d, a + off, b + off, idesc, k != 0);
  }
}
// D[128 x DT] (+)= A[128 x 128] B[128 x DT]: A 16-bit in tensor memory with its first 64 columns of K
// at a_lo and the other 64 at a_hi, B rows = K.
template <int DT>
__device__ __forceinline__ void mma_pb(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_smem, uint32_t idesc,
                                       bool accumulate) {
  const uint64_t b = ptx::smem_desc(kDescMN, b_smem);
#pragma unroll
  for (int k = 0; k < 8; ++k)
    mma_ts(d, (k < 4 ? a_lo : a_hi) + static_cast<uint32_t>((k % 4) * 8), b + static_cast<uint64_t>(k * 16 * 128 / 16),
           idesc, (accumulate || k != 0) ? 1u : 0u);
}

// Zero rows [first, 128) of an operand tile (one warp), before the MMA reads them.
template <int DT>
__device__ __forceinline__ void zero_rows(uint32_t tile, int first, int lane) {
#pragma unroll
  for (int j = 0; j < DT / 64; ++j)
    for (int i = first * 8 + lane; i < 128 * 8; i += 32)
      ptx::st_shared_v4(tile + j * kBoxBytes + i * 16, make_uint4(0, 0, 0, 0));
  ptx::fence_proxy_async_smem();
  __syncwarp();
}

// The tiles need a 1024-byte start, which is where dynamic shared memory begins when a kernel has no
// other; should that ever change, the call reports itself as failed instead of reading wrong tiles.
__device__ __forceinline__ bool aligned_start(const uint8_t* smem, int32_t* status) {
  const bool ok = (ptx::smem_u32(smem) & 1023u) == 0;
  if (!ok && threadIdx.x == 0 && status != nullptr) atomicOr(status, ST_LOAD);
  return ok;
}

template <typename T>
__host__ __device__ constexpr uint32_t mma_fmt() {
  return std::is_same<T, __half>::value ? 0u : 1u;
}

// One tile through the ring slot `dst`: rows from `valid` on are cleared before the consumers see it.
// Called by the whole load warp; returns false when a wait ran out.
template <int DT>
static __device__ __forceinline__ bool ring_load(uint32_t dst, const CUtensorMap* tm, int head, int token, int valid,
                                                 uint64_t* full, uint64_t* empty, uint32_t empty_parity, uint64_t* fix,
                                                 uint32_t* fix_phase, int lane, volatile int* cta_abort,
                                                 int32_t* status) {
  bool ok = true;
  const bool ragged = valid < kTile;
  if (lane == 0) {
    ok = ptx::mbar_wait(empty, empty_parity, cta_abort, status, ST_LOAD);
    if (ok) {
      uint64_t* bar = ragged ? fix : full;
      ptx::mbar_arrive_expect_tx(bar, (DT / 64) * kBoxBytes);
      load_tile<DT>(dst, tm, head, token, bar);
    }
  }
  ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
  if (ok && ragged) {
    // every lane waits for the copy itself: its stores to the tile have to come after it
    ok = warp_wait(fix, *fix_phase, cta_abort, status, ST_LOAD);
    if (!ok) return false;
    *fix_phase ^= 1u;
    zero_rows<DT>(dst, valid, lane);
    if (lane == 0) ptx::mbar_arrive(full);
  }
  return ok;
}

__device__ __forceinline__ void drain_copies() {
  const uint64_t t0 = ptx::globaltimer_ns();
  while (ptx::globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
}

// Results leave the accumulator 32 columns of a row per thread.  A thread's own stores would touch 32
// rows per instruction, about 2000 cycles a tile; a tile that lies inside its sequence goes to shared
// memory instead, where the operands were, and from there as one tile store.  (A tile that reaches past
// its sequence must not write there: its rows are stored one by one.)
// `lo_tile` / `lo_dst` (0 / null: none) take what rounding to 16 bits cut off, rounded in its turn.
template <typename T>
__device__ __forceinline__ void round_cols(const float (&v)[32], int g, float scale, uint4* hi, uint4* lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = v[g * 8 + 2 * e] * scale, b = v[g * 8 + 2 * e + 1] * scale;
    h[e] = pack2<T>(a, b);
    const T* r = reinterpret_cast<const T*>(&h[e]);
    l[e] = pack2<T>(a - Cvt<T>::to_f(r[0]), b - Cvt<T>::to_f(r[1]));
  }
  *hi = make_uint4(h[0], h[1], h[2], h[3]);
  *lo = make_uint4(l[0], l[1], l[2], l[3]);
}
template <typename T>
__device__ __forceinline__ void stage_cols(uint32_t taddr, uint32_t tile, uint32_t lo_tile, int row, int col0,
                                           float scale) {
  float v[32];
  tmem_ld32(taddr, v);
  tmem_wait_ld();
  const uint32_t at = (col0 / 64) * kBoxBytes + row * 128;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint4 hi, lo;
    round_cols<T>(v, g, scale, &hi, &lo);
    const uint32_t chunk = static_cast<uint32_t>((col0 % 64) / 8 + g) ^ (static_cast<uint32_t>(row) & 7u);
    ptx::st_shared_v4(tile + at + (chunk << 4), hi);
    if (lo_tile != 0) ptx::st_shared_v4(lo_tile + at + (chunk << 4), lo);
  }
}
template <typename T>
__device__ __forceinline__ void store_cols(uint32_t taddr, T* dst, T* lo_dst, int col0, int d, float scale,
                                           bool row_ok) {
  float v[32];
  tmem_ld32(taddr, v);
  tmem_wait_ld();
  if (!row_ok) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint4 hi, lo;
    round_cols<T>(v, g, scale, &hi, &lo);
    if (col0 + g * 8 >= d) continue;
    st_global_v4(dst + col0 + g * 8, hi);
    if (lo_dst != nullptr) st_global_v4(lo_dst + col0 + g * 8, lo);
  }
}
// 32 fp32 columns of a row to the same place of the CTA `peer` of the cluster, and those received added to
// this CTA's own.  The 16 bytes of neighbouring rows lie side by side.
__device__ __forceinline__ void send_cols(uint32_t taddr, uint32_t place, uint32_t peer) {
  float v[32];
  tmem_ld32(taddr, v);
  tmem_wait_ld();
  uint32_t there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(place), "r"(peer));
#pragma unroll
  for (int g = 0; g < 8; ++g)
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(there + g * 128 * 16), "f"(v[4 * g]),
                 "f"(v[4 * g + 1]), "f"(v[4 * g + 2]), "f"(v[4 * g + 3])
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void store_sum_cols(uint32_t taddr, uint32_t place, T* dst, int col0, int d, float scale,
                                               bool row_ok) {
  float v[32];
  tmem_ld32(taddr, v);
  tmem_wait_ld();
  if (!row_ok) return;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float r[8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(r[4 * h]), "=f"(r[4 * h + 1]), "=f"(r[4 * h + 2]), "=f"(r[4 * h + 3])
                   : "r"(place + (2 * g + h) * 128 * 16)
                   : "memory");
    uint32_t o[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
      o[e] = pack2<T>((v[g * 8 + 2 * e] + r[2 * e]) * scale, (v[g * 8 + 2 * e + 1] + r[2 * e + 1]) * scale);
    if (col0 + g * 8 < d) st_global_v4(dst + col0 + g * 8, make_uint4(o[0], o[1], o[2], o[3]));
  }
}
// After a warp has staged its part: say so, and (the one thread) wait for all and store the tile, and the
// second one unless lo_tile is 0.
template <int DT>
static __device__ __forceinline__ void store_tile(bool issuer, uint64_t* staged, uint32_t tile, const CUtensorMap* tm,
                                                  uint32_t lo_tile, const CUtensorMap* lo_tm, int head, int token,
                                                  int lane, volatile int* cta_abort, int32_t* status) {
  ptx::fence_proxy_async_smem();
  __syncwarp();
  if (lane == 0) ptx::mbar_arrive(staged);
  if (issuer && ptx::mbar_wait(staged, 0, cta_abort, status, ST_MATH)) {
#pragma unroll
    for (int j = 0; j < DT / 64; ++j) {
      tma_store_3d(tm, tile + j * kBoxBytes, j * 64, head, token);
      if (lo_tile != 0) tma_store_3d(lo_tm, lo_tile + j * kBoxBytes, j * 64, head, token);
    }
    ptx::bulk_commit_group();
    ptx::bulk_wait_group_read<0>();
  }
}

// What every kernel is told about one [tokens, heads, head_dim] tensor besides its tile map.
struct View {
  void* ptr;
  int64_t st, sh;  // element strides of a token and of a head
};

// fp16 has 40 powers of two for dS = P (dP - D): upstream gradients of 1e-4 and probabilities of a long row
// leave few of them above its last step.  dS is formed times 2^k such that the greatest value that it can
// have, 2 head_dim max|dO| max|V|, stays below 2^15; dQ and dK are scaled back in fp32.  The D kernel, which
// reads dO anyway, leaves one (max|dO|, max|V|) per block; infinities, NaN and rows behind the last sequence
// have no say.
constexpr int kMaxBounds = 2048;  // blocks of the D kernel

struct Params {
  Plan plan;
  int hq, hk, d, total;
  int gp, gp_shift, tq, nsub;  // packed heads, log2, tokens per tile, packed groups per kv head
  int gran;                    // index of the tile height that this kernel's items have
  float share;                 // dK, dV: plan's area per token of the longest below which key tiles are shared
  float scale, scale_log2;
  float* lse2;   // [hq][total] base-2 log-sum-exp of the scaled scores
  float* delta;  // [hq][total] dot(dO, O)
  View o, dq, dk, dv;
  void* o_lo;  // laid out as o
  const float2* bounds;  // fp16 backward: [n_bounds] (max|dO|, max|V|)
  int n_bounds;
  int32_t* status;
};

// The tensor-map encoder is a driver call and wants a current context: a thread that has made no runtime
// call yet (an autograd worker, say) gets its device's own.  Allowed during stream capture.
inline void bind_context() {
  int dev = 0;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaSetDevice(dev);
}

// Host side (attn_fwd.cu)
int fill_params(Params* p, const char* what, const int32_t* plan, int64_t batch, int64_t total, int64_t hq, int64_t hk,
                int64_t d, float scale, int dtype);
int check_view(const char* what, const void* p, int64_t st, int64_t sh, int heads, int64_t total);
int encode_rows(CUtensorMap* tm, const void* ptr, int dtype, int d, int heads, int64_t total, int64_t sh, int64_t st,
                int box_heads, int box_tokens, const char* what);

}  // namespace attn
}  // namespace bt
