// moe_mx_gemm.cu — the microscaled product on the block-scaled tensor cores,
// for one weight matrix or for one a run of rows (the experts' products):
//   out[t, n] = alpha[e] * sum_k A[t, k] SA[t, k / blk] * W[e, n, k] SW[e, n, k / blk]
// for the rows t of expert e, off[e] <= t < off[e + 1]. Products and block
// scales are applied by tcgen05.mma (exact), sums are fp32, the result is
// rounded once to the output's type. Rows outside the runs are not written.
//
// Weights are the M operand (128 rows a tile), tokens the N operand (16..256 a
// tile, chosen per call): a decode call then streams whole 128-row weight
// tiles against one narrow token tile, and a run's last tile issues only the
// columns it has.
//
// Warp roles (480 threads, one CTA per SM, persistent):
//   warp 0       TMA producer: 128 bytes of K of the weight tile and of the
//                token tile per stage (256 4-bit or 128 8-bit values)
//   warp 1       TMEM owner and MMA issuer: four K slices of 32 bytes a stage
//   warps 2-5    scale loaders, four stages at a time. Scales are stored row by
//                row; the tensor core wants, for 128 rows, word w of row r at
//                lane r % 32, column r / 32: a lane loads the words of rows
//                r, r + 32, r + 64, r + 96 and stores them transposed.
//   warps 6-13   epilogue: TMEM -> registers -> global, two warps a lane quarter
//   warp 14      copies of the stages' scales from shared memory to TMEM
//                (tcgen05.cp), where the MMA issuer does not do that itself
// TMEM (512 columns): two or four slots of scales at the top and two accumulators of
// the tile's width below, which overlap in their middle when two do not fit;
// the epilogue drains the shared columns first and frees them.
// Few tiles and a long K: a cluster of up to 8 CTAs splits K, and each adds its
// share of the tokens over the cluster's shared memory in rank order, so there
// is no scratch, no atomics, and one answer.
//
// What bounds it (B200, random values, back to back in a graph):
//   8192 x 7168 x 4096 nvfp4    107 us, 4.5 PFLOP/s: a stage takes 780 cycles
//     without any loads (87 us), where its four MMAs are 512: the twelve scale
//     copies and the issue of both do not hide behind them
//   8192 x 7168 x 4096 mxfp8    174 us, 2.8 PFLOP/s: the card's power limit
//   32 experts x 7168 x 4096 nvfp4, 64 rows   71 us, 6.3 TB/s: HBM (27 experts
//     with rows; 28 are 79 us, as their tiles are 6.05 waves of CTAs)
//   32 experts x 2048 x 7168 mxfp4, 8192 rows 87 us, 4.3 TB/s: eight stages a
//     tile, in which neither HBM (45% by its counter) nor the tensor pipe (34%) is kept busy;
//     the MMA issuer waits in turn for tiles, scales and accumulators
//   8 x 7168 x 4096 nvfp4       7.4 us: launch, one exchange across the
//     cluster and some 2.6 us of weights
#include <atomic>
#include <type_traits>

#include "moe_kernels.h"
#include "moe_mx.cuh"

namespace moe {

namespace {

constexpr int kMxMaxExperts = kMxGemmMaxExperts;
constexpr int kMxTileN = 128;     // weight rows of a tile
constexpr int kMxStageK = 128;    // bytes of K of a stage
constexpr int kMxGemmThreads = 480;
constexpr int kMxSfWarp0 = 2, kMxSfWarps = 4;
constexpr int kMxEpiWarp0 = 6, kMxEpiWarps = 8;
constexpr int kMxCopyWarp = 14;
constexpr uint64_t kMxWaitNs = 2000000000ull;  // 2 s: only reached if something is broken

__device__ unsigned g_mx_status;  // kErrTimeout if a bounded wait gave up

template <int kFmt, int kNT, bool kPair>
struct MxCfg {
  static constexpr int kW = kFmt == kFmtNvfp4 ? 4 : (kFmt == kFmtMxfp4 ? 2 : 1);  // scale words of a row and stage
  static constexpr int kChunks = kNT > 128 ? 2 : 1;                               // 128-token groups of scales
  static constexpr int kTileBytes = kMxTileN * kMxStageK;
  static constexpr int kStageBytes = kTileBytes + (kPair ? kNT / 2 : kNT) * kMxStageK;  // a pair halves the tokens
  static constexpr int kSfBytes = kW * 512 * (1 + kChunks);
  static constexpr int kStages = kPair ? (kW > 2 ? 4 : 5) : (kNT > 64 ? 5 : (kNT > 32 ? 6 : 8));
  static constexpr int kGroupBytes = 4 * kSfBytes;  // scales of four stages
  static constexpr int kGroups = kPair ? (kW > 2 ? 3 : 4) : 2;  // slots of them
  static constexpr int kSfCols = kW * 4 * (1 + kChunks);  // TMEM columns of one slot
  // The copies of scales to TMEM are issued by a warp of their own, up to four
  // stages ahead; among the MMAs, one warp's issue took 450 of the 950 cycles of
  // a stage. Not so for pairs with nvfp4, whose twelve copies a stage slow the
  // MMAs down when they run ahead of them. Measured, copies apart / in line:
  // experts' nvfp4 products of 64 rows 73.9 / 79.2 us, 8192 x 7168 x 4096 mxfp4
  // 95.8 / 97.3 us, mxfp8 182.8 / 184.5 us, nvfp4 112.8 / 107.0 us.
  static constexpr bool kCopyApart = !kPair || kW < 4;
  static constexpr int kSlots = kCopyApart ? 4 : 2;
  static constexpr int kAccCols = (512 - kSlots * kSfCols) & ~31;
  // 16-column pieces of the overlap of two widest accumulators that a warp of the epilogue holds
  static constexpr int kShared = kNT - ((kAccCols - kNT) & ~31);
  static constexpr int kHeld = kShared > 0 ? (kShared / 16 + 1) / 2 : 0;
  // a split's partial sums take the ring's place: its cluster has one tile, whose stages are used up by then
  static constexpr int kPartBytes = kNT * kMxTileN * 4;
  static constexpr size_t kSmem = 1024 + (size_t)kStages * kStageBytes + kGroups * kGroupBytes;
  static_assert(kPair || kPartBytes <= kStages * kStageBytes, "partial sums reuse the ring");
  static_assert(kSlots <= kStages, "the readers of a TMEM slot are known by the ring stage they free");
};

struct MxGemmArgs {
  const uint8_t* sa;   // [R][nsc]
  const uint8_t* sw;   // [E][N][nsc]
  const int32_t* off;  // [E + 1], or nullptr: one run of R rows
  const float* alpha;  // [E] or nullptr
  void* out;
  int64_t out_ld;
  int out_dt;
  int E, R, N;
  int nsc;             // scales of a row
  int nk;              // stages of K
  int tn;              // tokens of a tile (multiple of 16, <= kNT)
  int box;             // token rows of one copy
  int split;           // CTAs of a cluster, each with its share of K
};

struct __align__(16) MxCtl {
  uint64_t full[8], empty[8];                      // ring of operand tiles
  uint64_t sf_full[4], sf_empty[4], peer_sf[4];    // groups of scales; peer_sf: the second CTA's, by its relay
  uint64_t cp_full[4];                             // scales in TMEM
  uint64_t tfull[2], acc_free, peer_acc;           // accumulators
  uint64_t part_ready;                             // a split's partial sums
  uint64_t mma_done, cp_done;                      // after a wait that gave up
  uint32_t tmem_base;
  int abort_flag;
  int start[kMxMaxExperts + 1];   // first row of each run
  int count[kMxMaxExperts];       // rows of each run
  int prefix[kMxMaxExperts + 1];  // first token tile of each run
};

struct MxUnit {
  int e, n0, row0, cnt;
};

__device__ __forceinline__ MxUnit mx_unit(const MxCtl* c, const MxGemmArgs& p, int u, int ntn, int tile_rows) {
  MxUnit x;
  const int g = u / ntn;
  x.n0 = (u - g * ntn) * tile_rows;
  int lo = 0, hi = p.E - 1;
  while (lo < hi) {  // last run whose first tile is <= g (empty runs share prefixes)
    const int mid = (lo + hi + 1) >> 1;
    if (c->prefix[mid] <= g) lo = mid; else hi = mid - 1;
  }
  x.e = lo;
  const int j = (g - c->prefix[lo]) * p.tn;
  x.row0 = c->start[lo] + j;
  x.cnt = min(p.tn, c->count[lo] - j);
  return x;
}

__device__ __forceinline__ void mx_abort(MxCtl* c) {
  atomicOr(&g_mx_status, kErrTimeout);
  *reinterpret_cast<volatile int*>(&c->abort_flag) = 1;
}
__device__ __forceinline__ bool mx_aborted(MxCtl* c) { return *reinterpret_cast<volatile int*>(&c->abort_flag) != 0; }

// Both operands' maps have three dimensions (bytes of a row, rows, planes).
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// The same into this CTA's shared memory, counted on the barrier at `bar` (a
// cluster address): both CTAs of a pair count on the first one's.
__device__ __forceinline__ void tma_load_3d_pair(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
      : "memory");
}

// 32 rows x 16 bytes of shared memory (rows 16 bytes apart) to 4 TMEM columns
// of lanes 0-31, repeated in the other three lane quarters.
template <bool kPair>
__device__ __forceinline__ void tmem_cp_sf(uint32_t taddr, uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu);
  d |= static_cast<uint64_t>(128u >> 4) << 16;  // leading offset (one 16-byte column only: unused)
  d |= static_cast<uint64_t>(128u >> 4) << 32;  // 128 B between 8-row groups
  d |= static_cast<uint64_t>(1u) << 46;         // descriptor version, no swizzle
  if constexpr (kPair)  // in both CTAs, each from its own shared memory
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(d) : "memory");
}

// Instruction descriptor of the block-scaled kinds, A and B K-major, M = 128 (256 for a pair):
// scale id of B in [4,6), type of A in [7,10) and of B in [10,13) (e2m1 = 1 in
// the 4-bit kinds, e4m3 = 0 in mxf8f6f4), N >> 3 in [17,23), scale type bit 23
// (0 e4m3, 1 e8m0), M >> 7 in [27,29), scale id of A in [29,31). The scale id
// is the byte of the 32-bit scale word that holds the K slice's first scale.
template <int kFmt, bool kPair>
__device__ __forceinline__ uint32_t mx_idesc(int n, uint32_t id) {
  const uint32_t type = kFmt == kFmtMxfp8 ? 0u : 1u;
  const uint32_t scale = kFmt == kFmtNvfp4 ? 0u : 1u;
  return (id << 4) | (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (scale << 23) |
         ((kPair ? 2u : 1u) << 27) | (id << 29);
}

#define MX_MMA(GROUP, KIND)                                                                              \
  asm volatile(                                                                                         \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                                  \
      "tcgen05.mma.cta_group::" GROUP "." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),       \
      "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)                                            \
      : "memory")
template <int kFmt, bool kPair>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb,
                                       uint32_t acc) {
  if constexpr (kFmt == kFmtNvfp4) {
    if constexpr (kPair) MX_MMA("2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
    else MX_MMA("1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  } else if constexpr (kFmt == kFmtMxfp4) {
    if constexpr (kPair) MX_MMA("2", "kind::mxf4.block_scale.scale_vec::2X");
    else MX_MMA("1", "kind::mxf4.block_scale.scale_vec::2X");
  } else {
    if constexpr (kPair) MX_MMA("2", "kind::mxf8f6f4.block_scale.scale_vec::1X");
    else MX_MMA("1", "kind::mxf8f6f4.block_scale.scale_vec::1X");
  }
}
#undef MX_MMA

// The same on this CTA's barrier alone.
template <bool kPair>
__device__ __forceinline__ void mx_commit_own(uint64_t* bar) {
  if constexpr (kPair)
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
  else
    mma_commit(bar);
}

// Arrive on `bar` (of both CTAs of a pair) once this thread's earlier MMAs and copies are done.
template <bool kPair>
__device__ __forceinline__ void mx_commit(uint64_t* bar) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .b16 m;\n\tmov.b16 m, 3;\n\t"
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}" ::"r"(
            smem_u32(bar))
        : "memory");
  else
    mma_commit(bar);
}
template <bool kPair>
__device__ __forceinline__ void mx_tmem_alloc(uint32_t* dst) {
  if constexpr (kPair) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(dst)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    tmem_alloc(dst, 512);
    tmem_relinquish();
  }
}
template <bool kPair>
__device__ __forceinline__ void mx_tmem_dealloc(uint32_t taddr) {
  if constexpr (kPair)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
  else
    tmem_dealloc(taddr, 512);
}

// ---- cluster helpers --------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_map(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_arrive_remote(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ void cluster_arrive_remote_relaxed(uint32_t addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
__device__ __forceinline__ bool cluster_wait_bounded(uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
  const uint64_t t0 = global_timer_ns();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    if (ok) return true;
    if (global_timer_ns() - t0 > limit_ns) return false;
  }
}
__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}
// This CTA's barrier and, in a pair, the one that the second CTA's relay arrives on.
template <bool kPair>
__device__ __forceinline__ bool mx_wait_both(uint64_t* own, uint64_t* peer, uint32_t parity) {
  if (!mbar_wait_bounded(own, parity, kMxWaitNs)) return false;
  if constexpr (kPair) return cluster_wait_bounded(peer, parity, kMxWaitNs);
  return true;
}

__device__ __forceinline__ void epi_bar_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
static_assert(kMxEpiWarps * 32 == 256, "epi_bar_sync counts the epilogue's threads");

__device__ __forceinline__ void mx_out_store(const MxGemmArgs& p, int64_t row, int n, float v) {
  const int64_t i = row * p.out_ld + n;
  if (p.out_dt == kDtBf16)
    static_cast<__nv_bfloat16*>(p.out)[i] = __float2bfloat16_rn(v);
  else if (p.out_dt == kDtFp16)
    static_cast<__half*>(p.out)[i] = __float2half_rn(v);
  else
    static_cast<float*>(p.out)[i] = v;
}

// Weight row n of `cnt` tokens (at most 16) from row `row` on. The type is
// decided once for all of them, not for each: 0.5 to 1% of a call of 1000 rows or more.
template <typename T, typename F>
__device__ __forceinline__ void mx_out_column(T* o, int64_t ld, int cnt, const float (&v)[16], float alpha, F round) {
#pragma unroll
  for (int j = 0; j < 16; ++j, o += ld)
    if (j < cnt) *o = round(v[j] * alpha);
}
__device__ __forceinline__ void mx_out_column(const MxGemmArgs& p, int64_t row, int n, int cnt, const float (&v)[16], float alpha) {
  const int64_t i = row * p.out_ld + n;
  if (p.out_dt == kDtBf16)
    mx_out_column(static_cast<__nv_bfloat16*>(p.out) + i, p.out_ld, cnt, v, alpha, [](float x) { return __float2bfloat16_rn(x); });
  else if (p.out_dt == kDtFp16)
    mx_out_column(static_cast<__half*>(p.out) + i, p.out_ld, cnt, v, alpha, [](float x) { return __float2half_rn(x); });
  else
    mx_out_column(static_cast<float*>(p.out) + i, p.out_ld, cnt, v, alpha, [](float x) { return x; });
}

// The scale words of one row and stage, kA bytes a load (rows and base are
// aligned to kA); `left` scales remain in the row, none or less: zeros. Rows
// that are whole stages, the usual ones, take one load, skipped where there is
// nothing. Of several loads, those past the end go to `safe`, and
// `word` below drops what they bring: a branch around each took some hundred cycles.
template <int kW, int kA>
__device__ __forceinline__ void mx_sf_aligned(const uint8_t* s, int left, const uint8_t* safe, uint32_t* w) {
  constexpr bool kWhole = kA == 4 * kW;
  if (kWhole) {
#pragma unroll
    for (int i = 0; i < kW; ++i) w[i] = 0;
    if (left <= 0) return;
  }
#pragma unroll
  for (int i = 0; i < 4 * kW; i += kA) {
    const uint8_t* q = kWhole || i < left ? s + i : safe;
    uint32_t* d = w + i / 4;
    // volatile: the loads stay before the wait for the slot
    if constexpr (kA == 16)
      asm volatile("ld.global.nc.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3]) : "l"(q));
    else if constexpr (kA == 8)
      asm volatile("ld.global.nc.v2.u32 {%0, %1}, [%2];" : "=r"(d[0]), "=r"(d[1]) : "l"(q));
    else
      asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(d[0]) : "l"(q));
  }
}

// Rows of any length: the kW + 1 aligned words around the bytes, shifted into
// place by mx_sf_shift. `inside`: all of them lie in the tensor; otherwise the
// words are put together from those bytes that lie in [begin, end).
template <int kW>
__device__ __forceinline__ void mx_sf_around(const uint8_t* s, int left, bool inside, const uint8_t* begin,
                                             const uint8_t* end, uint32_t* v) {
  if (inside) {
    const uint8_t* a = left > 0 ? s - (reinterpret_cast<uintptr_t>(s) & 3u) : begin;
#pragma unroll
    for (int i = 0; i <= kW; ++i) asm volatile("ld.global.nc.u32 %0, [%1];" : "=r"(v[i]) : "l"(a + 4 * i));
  } else {
    const uint8_t* a = s - (reinterpret_cast<uintptr_t>(s) & 3u);
#pragma unroll
    for (int i = 0; i <= kW; ++i) {
      v[i] = 0;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint8_t* q = a + 4 * i + b;
        if (left > 0 && q >= begin && q < end) v[i] |= static_cast<uint32_t>(__ldg(q)) << (8 * b);
      }
    }
  }
}
// Word i of a row's stage from the words around it; scales past the row's end are 0.
__device__ __forceinline__ uint32_t mx_sf_shift(const uint32_t* v, int i, int off, int left) {
  const uint32_t w = __funnelshift_r(v[i], v[i + 1], 8 * off);
  const int keep = left - 4 * i;  // bytes of this word that belong to the row
  return keep >= 4 ? w : (keep > 0 ? w & (0xFFFFFFFFu >> (8 * (4 - keep))) : 0u);
}

// A bounded wait gives up for the whole warp or for none of it.
__device__ __forceinline__ bool all_lanes(bool ok) { return __all_sync(0xffffffffu, ok); }

__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}

template <int kFmt, int kNT, bool kPair>
__global__ void __launch_bounds__(kMxGemmThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                   const MxGemmArgs p) {
  using Cfg = MxCfg<kFmt, kNT, kPair>;
  constexpr int kS = Cfg::kStages, kW = Cfg::kW;
  extern __shared__ uint8_t smem_raw[];
  __shared__ MxCtl ctl_;
  MxCtl* ctl = &ctl_;
  uint8_t* tiles = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
  uint8_t* sfs = tiles + kS * Cfg::kStageBytes;
  float* part = reinterpret_cast<float*>(tiles);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  // a unit is one tile of weight rows x tokens, and belongs to a cluster: a
  // pair (256 weight rows, 128 a CTA) or `split` CTAs along K (1: no cluster)
  const bool clustered = kPair || p.split > 1;
  const int members = kPair ? 2 : p.split;
  constexpr int kTileRows = kPair ? 2 * kMxTileN : kMxTileN;
  const int ntn = (p.N + kTileRows - 1) / kTileRows;
  const int rank = clustered ? blockIdx.x % members : 0;
  const int u_first = blockIdx.x / members, u_step = gridDim.x / members;
  const int k0 = kPair ? 0 : static_cast<int>((static_cast<int64_t>(p.nk) * rank) / p.split);
  const int k1 = kPair ? p.nk : static_cast<int>((static_cast<int64_t>(p.nk) * (rank + 1)) / p.split);
  const int my_n = kPair ? rank * kMxTileN : 0;  // first weight row of this CTA inside the tile

  if (tid == 0) {
    for (int s = 0; s < kS; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 1);
    }
    for (int b = 0; b < Cfg::kGroups; ++b) {
      mbar_init(&ctl->sf_full[b], kMxSfWarps);
      mbar_init(&ctl->peer_sf[b], 1);
      mbar_init(&ctl->sf_empty[b], 1);
    }
    mbar_init(&ctl->tfull[0], 1);
    mbar_init(&ctl->tfull[1], 1);
    mbar_init(&ctl->acc_free, kMxEpiWarps);
    mbar_init(&ctl->peer_acc, kMxEpiWarps);
    mbar_init(&ctl->part_ready, p.split);
    mbar_init(&ctl->mma_done, 1);
    mbar_init(&ctl->cp_done, 1);
    for (int b = 0; b < Cfg::kSlots; ++b) mbar_init(&ctl->cp_full[b], 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
    prefetch_tensormap(&map_w);
    prefetch_tensormap(&map_a);
  }
  if (warp == 1) {
    mx_tmem_alloc<kPair>(&ctl->tmem_base);
  }
  griddep_wait();
  griddep_launch_dependents();
  // Runs and their token tiles: one warp, 32 experts at a time. Bounds are kept
  // inside [0, R] and made not to decrease, so that the runs are disjoint
  // whatever the offsets hold.
  if (!p.off) {
    if (tid == 64) {
      ctl->start[0] = 0;
      ctl->count[0] = p.R;
      ctl->prefix[0] = 0;
      ctl->prefix[1] = (p.R + p.tn - 1) / p.tn;
    }
  } else if (warp == 2) {
    int tiles = 0, from = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + lane;
      int lo = from, hi = from;
      if (e < p.E) {
        lo = min(max(__ldg(p.off + e), from), p.R);
        hi = min(max(__ldg(p.off + e + 1), lo), p.R);
      }
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {  // running maximum of the ends
        const int v = __shfl_up_sync(0xffffffffu, hi, o);
        if (lane >= o) hi = max(hi, v);
      }
      const int before = __shfl_up_sync(0xffffffffu, hi, 1);
      if (lane > 0) lo = max(lo, before);
      const int t = (hi - lo + p.tn - 1) / p.tn;
      int inc = t;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      if (e < p.E) {
        ctl->start[e] = lo;
        ctl->count[e] = hi - lo;
        ctl->prefix[e] = tiles + inc - t;
      }
      tiles += __shfl_sync(0xffffffffu, inc, 31);
      from = __shfl_sync(0xffffffffu, hi, 31);
    }
    if (lane == 0) ctl->prefix[p.E] = tiles;
  }
  tc_fence_before();
  if (clustered)
    cluster_sync_all();  // the barriers of every CTA of the cluster are set up
  else
    __syncthreads();
  tc_fence_after();
  const int units = ctl->prefix[p.E] * ntn;
  const uint32_t tmem = ctl->tmem_base;
  const int acc1 = (Cfg::kAccCols - p.tn) & ~31;  // first column of the second accumulator
  const uint32_t acc_at[2] = {tmem, tmem + acc1};
  const uint32_t sf_at = tmem + Cfg::kAccCols;

  // Issues the copies of a stage's scales (stage kg of group slot gs) to TMEM slot `slot`.
  const auto copy_scales = [&](uint32_t gs, int kg, uint32_t slot, int cnt) {
    const uint32_t sf = smem_u32(sfs + gs * Cfg::kGroupBytes + kg * Cfg::kSfBytes);
    const uint32_t t_w = sf_at + slot * Cfg::kSfCols, t_a = t_w + 4 * kW;
#pragma unroll
    for (int i = 0; i < kW; ++i) {
      tmem_cp_sf<kPair>(t_w + 4 * i, sf + i * 512);
#pragma unroll
      for (int c = 0; c < Cfg::kChunks; ++c)
        if (c * 128 < cnt)
          tmem_cp_sf<kPair>(t_a + (i * Cfg::kChunks + c) * 4, sf + kW * 512 + (i * Cfg::kChunks + c) * 512);
    }
  };
  // Waits for the scales of group `grp` and, from the kSlots-th stage on, for
  // the TMEM slot of stage `it` (its last readers: the MMAs kSlots stages back).
  const auto copy_ready = [&](uint32_t it, uint32_t grp, bool first) {
    bool ok = true;
    if (first)
      ok = mx_wait_both<kPair>(&ctl->sf_full[grp % Cfg::kGroups], &ctl->peer_sf[grp % Cfg::kGroups], (grp / Cfg::kGroups) & 1u);
    if (ok && it >= Cfg::kSlots)
      ok = mbar_wait_bounded(&ctl->empty[(it - Cfg::kSlots) % kS], ((it - Cfg::kSlots) / kS) & 1u, kMxWaitNs);
    return all_lanes(ok);
  };

  if (warp == 0) {
    // ======================= TMA producer =======================
    // The whole warp walks the loop and one elected lane issues (see the MMA
    // issuer); from a branch on the lane a copy takes some 200 cycles. Where the
    // MMA issuer is the slower one all the same, one lane does better: 8192 x
    // 7168 x 4096 nvfp4 107.3 against 110.9 us, mxfp8 182.6 against 174.2 us,
    // 1000 x 2048 x 7168 mxfp8 19.8 against 18.7 us.
    constexpr bool kWhole = Cfg::kCopyApart;
    uint32_t it = 0;
    const bool el = kWhole ? elect_one() : lane == 0;
    if (kWhole || el) {
      for (int u = u_first; u < units && !mx_aborted(ctl); u += u_step) {
        const MxUnit x = mx_unit(ctl, p, u, ntn, kTileRows);
        // token rows of this CTA: the columns that are issued, of which the
        // second CTA of a pair holds the second half
        const int rows_a = (x.cnt + 15) / 16 * (kPair ? 8 : 16);
        const int row_a = x.row0 + (kPair ? rank * rows_a : 0);
        const int boxes = (rows_a + p.box - 1) / p.box;
        const uint32_t bytes = Cfg::kTileBytes + boxes * p.box * kMxStageK;
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % kS;
          bool ok = mbar_wait_bounded(&ctl->empty[s], ((it / kS) & 1u) ^ 1u, kMxWaitNs);
          if (kWhole) ok = all_lanes(ok);
          if (!ok) { mx_abort(ctl); break; }
          if (el) {
            uint8_t* st = tiles + s * Cfg::kStageBytes;
            if constexpr (kPair) {
              // both CTAs' copies count on the first CTA's barrier
              const uint32_t bar = cluster_map(smem_u32(&ctl->full[s]), 0);
              if (rank == 0) mbar_arrive_expect_tx(&ctl->full[s], 2 * bytes);
              tma_load_3d_pair(st, &map_w, k * kMxStageK, x.n0 + my_n, x.e, bar);
              for (int b = 0; b < boxes; ++b)
                tma_load_3d_pair(st + Cfg::kTileBytes + b * p.box * kMxStageK, &map_a, k * kMxStageK, row_a + b * p.box, 0, bar);
            } else {
              mbar_arrive_expect_tx(&ctl->full[s], bytes);
              tma_load_3d(st, &map_w, k * kMxStageK, x.n0, x.e, &ctl->full[s]);
              for (int b = 0; b < boxes; ++b)
                tma_load_3d(st + Cfg::kTileBytes + b * p.box * kMxStageK, &map_a, k * kMxStageK, row_a + b * p.box, 0, &ctl->full[s]);
            }
          }
          if (kWhole) __syncwarp();
        }
      }
    }
    if (mx_aborted(ctl) && el) {
      // wait (bounded) for the copies in flight; the second CTA of a pair,
      // whose copies count elsewhere, gives them a millisecond
      if (rank == 0 || !kPair) {
        for (uint32_t j = it > (uint32_t)kS ? it - kS : 0; j < it; ++j)
          mbar_wait_bounded(&ctl->full[j % kS], (j / kS) & 1u, kMxWaitNs);
      } else {
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000) __nanosleep(1000);
      }
    }
  } else if (warp == 1) {
    // ======================= MMA issuer =======================
    // The whole warp walks the loop and one elected lane issues: with every
    // operand the same in all lanes an issue costs some 25 cycles, where a
    // branch on the lane cost some 70 for each (182 -> 145 us at 8192 x 7168 x 4096 nvfp4).
    if (!kPair || rank == 0) {
      uint32_t it = 0, tile = 0, grp = 0;
      const bool el = elect_one();
      for (int u = u_first; u < units && !mx_aborted(ctl); u += u_step, ++tile) {
        const MxUnit x = mx_unit(ctl, p, u, ntn, kTileRows);
        const int nmma = (x.cnt + 15) & ~15;
        const uint32_t d = acc_at[tile & 1u];
        // the tile before last has left this accumulator and the last one the columns they share
        if (tile > 0 && !all_lanes(mx_wait_both<kPair>(&ctl->acc_free, &ctl->peer_acc, (tile - 1) & 1u))) {
          mx_abort(ctl);
          break;
        }
        for (int k = k0; k < k1; ++k, ++it) {
          const int s = it % kS, kg = (k - k0) & 3;
          const bool group_ends = kg == 3 || k == k1 - 1;
          if constexpr (!Cfg::kCopyApart) {
            if (!copy_ready(it, grp, kg == 0)) { mx_abort(ctl); break; }
          }
          bool ok = mbar_wait_bounded(&ctl->full[s], (it / kS) & 1u, kMxWaitNs);
          if constexpr (Cfg::kCopyApart)
            ok = ok && mbar_wait_bounded(&ctl->cp_full[it % Cfg::kSlots], (it / Cfg::kSlots) & 1u, kMxWaitNs);
          if (!all_lanes(ok)) { mx_abort(ctl); break; }
          tc_fence_after();
          if (el) {
            if constexpr (!Cfg::kCopyApart) copy_scales(grp % Cfg::kGroups, kg, it % Cfg::kSlots, x.cnt);
            const uint32_t t_w = sf_at + (it % Cfg::kSlots) * Cfg::kSfCols, t_a = t_w + 4 * kW;
            const uint32_t st = smem_u32(tiles + s * Cfg::kStageBytes);
            const uint64_t dw = smem_desc_sw128(st), da = smem_desc_sw128(st + Cfg::kTileBytes);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              // slice j's scales: all four bytes of word j (nvfp4), half j % 2 of word j / 2 (mxfp4), byte j (mxfp8)
              const int word = kFmt == kFmtNvfp4 ? j : (kFmt == kFmtMxfp4 ? j / 2 : 0);
              const uint32_t id = kFmt == kFmtNvfp4 ? 0u : (kFmt == kFmtMxfp4 ? 2u * (j % 2) : j);
              mx_mma<kFmt, kPair>(d, dw + 2 * j, da + 2 * j, mx_idesc<kFmt, kPair>(nmma, id), t_w + 4 * word,
                                  t_a + word * Cfg::kChunks * 4, (k > k0 || j > 0) ? 1u : 0u);
            }
            mx_commit<kPair>(&ctl->empty[s]);
            if (!Cfg::kCopyApart && group_ends) mx_commit<kPair>(&ctl->sf_empty[grp % Cfg::kGroups]);
          }
          __syncwarp();
          if (group_ends) ++grp;
        }
        if (mx_aborted(ctl)) break;
        if (el) mx_commit<kPair>(&ctl->tfull[tile & 1u]);
        __syncwarp();
      }
      if (mx_aborted(ctl) && it > 0) {
        if (el) mx_commit<kPair>(&ctl->mma_done);
        mbar_wait_bounded(&ctl->mma_done, 0, kMxWaitNs);
      }
    } else {
      // The second CTA's relay: its scale loaders arrive on barriers of their
      // own CTA, and this warp passes that on to the first CTA. A release at
      // cluster scope takes some 1400 cycles here; in the scale loaders it
      // held up every group (120 -> 111 us at 8192 x 7168 x 4096 nvfp4).
      uint32_t grp = 0;
      bool ok = true;
      for (int u = u_first; u < units && ok && !mx_aborted(ctl); u += u_step) {
        for (int k = k0; k < k1; k += 4, ++grp) {
          const uint32_t gs = grp % Cfg::kGroups;
          ok = all_lanes(mbar_wait_bounded(&ctl->sf_full[gs], (grp / Cfg::kGroups) & 1u, kMxWaitNs));
          if (!ok) break;
          if (lane == 0) cluster_arrive_remote(cluster_map(smem_u32(&ctl->peer_sf[gs]), 0));
        }
      }
      if (!ok) mx_abort(ctl);
    }
  } else if (warp < kMxSfWarp0 + kMxSfWarps) {
    // ======================= scale loaders =======================
    // Four stages at a time into the next slot (of two, three or four): lane 8 j + r of warp b
    // loads stage j's words of rows 8 b + r, + 32, + 64, + 96 of every
    // 128-row group (four lanes read a row's neighbouring words) and stores
    // each word's four rows as one 16-byte piece.
    const int r0 = (warp - kMxSfWarp0) * 8 + (lane & 7), j = lane >> 3;
    const uint64_t low =
        reinterpret_cast<uint64_t>(p.sw) | reinterpret_cast<uint64_t>(p.sa) | static_cast<uint64_t>(p.nsc);
    const uint8_t* end_w = p.sw + static_cast<int64_t>(p.E) * p.N * p.nsc;
    const uint8_t* end_a = p.sa + static_cast<int64_t>(p.R) * p.nsc;
    // one loop for each kind of row, so that there are no branches among the loads
    const auto loop = [&](auto align) {
      constexpr int kA = decltype(align)::value;  // bytes of a load; 1: words around the bytes
      constexpr int kR = kA > 1 ? kW : kW + 1;    // words held of a row and stage
      const int64_t ld = p.nsc;
      // the words of stages k .. k + 3 of unit x: 128-row group g = 0 is the
      // weights', the others the tokens'
      const auto load = [&](const MxUnit& x, int k, uint32_t (&w)[1 + Cfg::kChunks][4][kR]) {
        const int n0 = x.n0 + my_n;
        const int at = (k + j) * 4 * kW;
        const int left = k + j < k1 ? p.nsc - at : 0;
        const uint8_t* base[2] = {p.sw + (static_cast<int64_t>(x.e) * p.N + n0) * ld, p.sa + x.row0 * ld};
        bool inside = true;
        if constexpr (kA == 1) {
          // the four stages' words of the last row of either side
          const int64_t last = static_cast<int64_t>(k + 4) * 4 * kW + 4;
          inside = (reinterpret_cast<uint64_t>(p.sw) & 3) == 0 && (reinterpret_cast<uint64_t>(p.sa) & 3) == 0 &&
                   base[0] + (min(kMxTileN, p.N - n0) - 1) * ld + last <= end_w && base[1] + (x.cnt - 1) * ld + last <= end_a;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int g = 0; g <= Cfg::kChunks; ++g) {
            const int r = r0 + 32 * q + (g > 1 ? 128 : 0);
            const int mine = r < (g == 0 ? p.N - n0 : x.cnt) ? left : 0;
            const uint8_t* s = base[g > 0] + r * ld + at;
            if constexpr (kA > 1)
              mx_sf_aligned<kW, kA>(s, mine, g == 0 ? p.sw : p.sa, w[g][q]);
            else
              mx_sf_around<kW>(s, mine, inside, g == 0 ? p.sw : p.sa, g == 0 ? end_w : end_a, w[g][q]);
          }
        }
      };
      // word i of row q of group g, of the stage that this lane loaded
      const auto word = [&](const MxUnit& x, int k, const uint32_t (&w)[1 + Cfg::kChunks][4][kR], int g, int q, int i) {
        if constexpr (kA == 4 * kW) return w[g][q][i];
        const int r = r0 + 32 * q + (g > 1 ? 128 : 0), at = (k + j) * 4 * kW;
        const int left = k + j < k1 && r < (g == 0 ? p.N - x.n0 - my_n : x.cnt) ? p.nsc - at : 0;
        if constexpr (kA > 1) {
          return 4 * i < left ? w[g][q][i] : 0u;
        } else {
          const uint8_t* b = g == 0 ? p.sw + (static_cast<int64_t>(x.e) * p.N + x.n0 + my_n) * ld : p.sa + x.row0 * ld;
          return mx_sf_shift(w[g][q], i, static_cast<int>((reinterpret_cast<uint64_t>(b) + r * ld + at) & 3u), left);
        }
      };
      uint32_t grp = 0;
      // words of stages k .. k + 3 into the next slot
      const auto put = [&](const MxUnit& x, int k, const uint32_t (&w)[1 + Cfg::kChunks][4][kR]) {
        const uint32_t gs = grp % Cfg::kGroups;
        if (!all_lanes(mbar_wait_bounded(&ctl->sf_empty[gs], ((grp / Cfg::kGroups) & 1u) ^ 1u, kMxWaitNs))) {
          mx_abort(ctl);
          return false;
        }
        uint8_t* sf = sfs + gs * Cfg::kGroupBytes + j * Cfg::kSfBytes + r0 * 16;
#pragma unroll
        for (int i = 0; i < kW; ++i) {
#pragma unroll
          for (int g = 0; g <= Cfg::kChunks; ++g)
            *reinterpret_cast<uint4*>(sf + (g == 0 ? i : kW + i * Cfg::kChunks + g - 1) * 512) =
                make_uint4(word(x, k, w, g, 0, i), word(x, k, w, g, 1, i), word(x, k, w, g, 2, i), word(x, k, w, g, 3, i));
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->sf_full[gs]);
        ++grp;
        return true;
      };
      if (kPair || clustered) {
        uint32_t w[1 + Cfg::kChunks][4][kR];
        bool ok = true;
        for (int u = u_first; u < units && ok && !mx_aborted(ctl); u += u_step) {
          const MxUnit x = mx_unit(ctl, p, u, ntn, kTileRows);
          for (int k = k0; k < k1 && ok; k += 4) {
            load(x, k, w);  // under way while the slot is still being read
            ok = put(x, k, w);
          }
        }
      } else if (u_first < units) {
        // A CTA by itself streams weights, whose scales come from HBM: the next
        // group's loads start before this one's are waited for. 32 experts x
        // 7168 x 4096 nvfp4, 64 rows on 27 of them: 74.2 -> 70.9 us; the longer code costs
        // calls of 8 and of 128 rows 1 to 2%. (A split has a group or two and loses 4%.
        // In a pair two groups of nvfp4 are 96 words a lane, which do not fit the
        // registers; mxfp4's 48 and mxfp8's 24 would, and were not tried.)
        MxUnit xa = mx_unit(ctl, p, u_first, ntn, kTileRows), xb = xa;
        int u = u_first, ka = k0, kb = k0;
        uint32_t wa[1 + Cfg::kChunks][4][kR], wb[1 + Cfg::kChunks][4][kR];
        // the group behind (x, k): false where there is none
        const auto next = [&](const MxUnit& x, int k, MxUnit& y, int& l) {
          y = x;
          l = k + 4;
          if (l < k1) return true;
          l = k0;
          u += u_step;
          if (u >= units || mx_aborted(ctl)) return false;
          y = mx_unit(ctl, p, u, ntn, kTileRows);
          return true;
        };
        load(xa, ka, wa);
        while (true) {
          bool more = next(xa, ka, xb, kb);
          if (more) load(xb, kb, wb);
          if (!put(xa, ka, wa) || !more) break;
          more = next(xb, kb, xa, ka);
          if (more) load(xa, ka, wa);
          if (!put(xb, kb, wb) || !more) break;
        }
      }
    };
    if (kW == 4 && (low & 15) == 0)
      loop(std::integral_constant<int, kW == 4 ? 16 : 4>{});
    else if (kW >= 2 && (low & 7) == 0)
      loop(std::integral_constant<int, kW >= 2 ? 8 : 4>{});
    else if ((low & 3) == 0)
      loop(std::integral_constant<int, 4>{});
    else
      loop(std::integral_constant<int, 1>{});
  } else if (warp == kMxCopyWarp) {
    // ======================= scale copies to TMEM =======================
    if (Cfg::kCopyApart && (!kPair || rank == 0)) {
      uint32_t it = 0, grp = 0;
      const bool el = elect_one();
      for (int u = u_first; u < units && !mx_aborted(ctl); u += u_step) {
        const MxUnit x = mx_unit(ctl, p, u, ntn, kTileRows);
        for (int k = k0; k < k1; ++k, ++it) {
          const int kg = (k - k0) & 3;
          const bool group_ends = kg == 3 || k == k1 - 1;
          if (!copy_ready(it, grp, kg == 0)) { mx_abort(ctl); break; }
          tc_fence_after();
          if (el) {
            copy_scales(grp % Cfg::kGroups, kg, it % Cfg::kSlots, x.cnt);
            mx_commit_own<kPair>(&ctl->cp_full[it % Cfg::kSlots]);
            if (group_ends) mx_commit<kPair>(&ctl->sf_empty[grp % Cfg::kGroups]);
          }
          __syncwarp();
          if (group_ends) ++grp;
        }
      }
      if (mx_aborted(ctl) && it > 0) {
        if (el) mx_commit<kPair>(&ctl->cp_done);
        mbar_wait_bounded(&ctl->cp_done, 0, kMxWaitNs);
      }
    }
  } else {
    // ======================= epilogue (8 warps) =======================
    const int q = warp & 3, half = (warp - kMxEpiWarp0) >> 2;
    const uint32_t t_lane = static_cast<uint32_t>(q * 32) << 16;
    const int etid = tid - kMxEpiWarp0 * 32;
    const int nl = q * 32 + lane;  // weight row of this thread inside the tile
    const int nch = p.tn / 16;
    const int shared_cols = p.tn - acc1;
    const int ovc = shared_cols > 0 ? (shared_cols + 15) / 16 : 0;
    uint32_t tile = 0;
    for (int u = u_first; u < units && !mx_aborted(ctl); u += u_step, ++tile) {
      const MxUnit x = mx_unit(ctl, p, u, ntn, kTileRows);
      const uint32_t buf = tile & 1u;
      const float alpha = p.alpha ? __ldg(p.alpha + x.e) : 1.0f;
      if (!all_lanes(mbar_wait_bounded(&ctl->tfull[buf], (tile >> 1) & 1u, kMxWaitNs))) { mx_abort(ctl); break; }
      __syncwarp();
      tc_fence_after();
      // buffer 0 shares its last columns with buffer 1's first: those go to
      // registers and are given back before anything is stored
      const auto column = [&](int i) { return (buf == 0 ? nch - 1 - i : i) * 16; };
      const auto store = [&](int c, const float (&v)[16]) {
        if (p.split > 1) {
#pragma unroll
          for (int j = 0; j < 16; ++j) part[(c + j) * kMxTileN + nl] = v[j];
        } else if (x.n0 + my_n + nl < p.N) {
          mx_out_column(p, static_cast<int64_t>(x.row0) + c, x.n0 + my_n + nl, x.cnt - c, v, alpha);
        }
      };
      float head[Cfg::kHeld > 0 ? Cfg::kHeld : 1][16];
#pragma unroll
      for (int h = 0; h < Cfg::kHeld; ++h) {
        const int i = half + 2 * h;
        if (i < ovc && column(i) < x.cnt) tmem_ld_32x32b_x16(acc_at[buf] + t_lane + column(i), head[h]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (!kPair || rank == 0)
          mbar_arrive(&ctl->acc_free);
        else  // nothing in memory to publish: the loads from TMEM are complete
          cluster_arrive_remote_relaxed(cluster_map(smem_u32(&ctl->peer_acc), 0));
      }
#pragma unroll
      for (int h = 0; h < Cfg::kHeld; ++h) {
        const int i = half + 2 * h;
        if (i < ovc && column(i) < x.cnt) store(column(i), head[h]);
      }
      for (int i = half + (ovc > half ? (ovc - half + 1) / 2 * 2 : 0); i < nch; i += 2) {
        const int c = column(i);
        if (c >= x.cnt) continue;
        float v[16];
        tmem_ld_32x32b_x16(acc_at[buf] + t_lane + c, v);
        store(c, v);
      }
      if (p.split > 1) {
        epi_bar_sync();
        if (etid < p.split) cluster_arrive_remote(cluster_map(smem_u32(&ctl->part_ready), etid));
        if (!all_lanes(cluster_wait_bounded(&ctl->part_ready, 0, kMxWaitNs))) { mx_abort(ctl); break; }
        // tokens rank, rank + split, ...: a warp a token, four weight rows a lane
        const int n = x.n0 + lane * 4;
        for (int t = rank + (warp - kMxEpiWarp0) * p.split; t < x.cnt; t += kMxEpiWarps * p.split) {
          const uint32_t at = smem_u32(part + t * kMxTileN + lane * 4);
          float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
          for (int r = 0; r < p.split; ++r) {
            const float4 v = ld_cluster_f4(cluster_map(at, r));
            sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
          }
          const int64_t row = static_cast<int64_t>(x.row0) + t;
          if (n < p.N) mx_out_store(p, row, n, sum.x * alpha);
          if (n + 1 < p.N) mx_out_store(p, row, n + 1, sum.y * alpha);
          if (n + 2 < p.N) mx_out_store(p, row, n + 2, sum.z * alpha);
          if (n + 3 < p.N) mx_out_store(p, row, n + 3, sum.w * alpha);
        }
      }
    }
  }

  tc_fence_before();
  __syncwarp();
  if (clustered)
    cluster_sync_all();  // no CTA leaves while another may use its shared memory or TMEM
  else
    __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    mx_tmem_dealloc<kPair>(tmem);
  }
}

template <int kFmt, int kNT, bool kPair>
cudaError_t mx_gemm_launch(const CUtensorMap& mw, const CUtensorMap& ma, const MxGemmArgs& p, int grid, cudaStream_t s) {
  using Cfg = MxCfg<kFmt, kNT, kPair>;
  static_assert(Cfg::kSmem + sizeof(MxCtl) <= 232448, "shared memory of a CTA");
  // the shared-memory opt-in is an attribute of the function on a device: one bit per device that has it
  static std::atomic<uint64_t> configured{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (!(configured.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(mx_gemm_kernel<kFmt, kNT, kPair>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(Cfg::kSmem));
    if (e != cudaSuccess) return e;
    configured.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kMxGemmThreads);
  cfg.dynamicSmemBytes = Cfg::kSmem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = kPair ? 2 : p.split;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kPair || p.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, mx_gemm_kernel<kFmt, kNT, kPair>, mw, ma, p);
}

template <int kFmt>
cudaError_t mx_gemm_launch_nt(const MxPlan& pl, const CUtensorMap& mw, const CUtensorMap& ma, const MxGemmArgs& p,
                              cudaStream_t s) {
  if (pl.pair) return mx_gemm_launch<kFmt, 256, true>(mw, ma, p, pl.grid, s);
  switch (pl.nt) {
    case 32: return mx_gemm_launch<kFmt, 32, false>(mw, ma, p, pl.grid, s);
    case 64: return mx_gemm_launch<kFmt, 64, false>(mw, ma, p, pl.grid, s);
    default: return mx_gemm_launch<kFmt, 128, false>(mw, ma, p, pl.grid, s);
  }
}

}  // namespace

// Tokens of a tile, K split and grid of a call.
//
// One run of rows: up to 64 rows are one tile. Beyond that the width with the
// least cost in rows loaded: waves of CTAs (or pairs, above 128 tokens) x
// stages x (weight rows + tokens), and for a split what its exchange takes,
// measured as some 800 + 6 a token. Checked against fixed widths of 64 to 256
// at 128 to 2048 x 7168 x 4096 nvfp4 and 1000 x 2048 x 7168 mxfp8: within 3% of
// the best one each time, where the worst took 1.6 to 2.6 times as long.
// Several runs, whose lengths only the device knows: by their mean length. 32
// x 7168 x 4096 nvfp4: at a mean of 32 rows tiles of 64 take 94 us and pairs of
// 256 102 us, at 64 rows 142 and 104 us, at 128 rows tiles of 128 149 us and
// pairs 111 us. All of even runs over many weight rows; the rule knows neither
// N nor the number of tiles. Few experts with small N get pairs that leave most
// SMs idle, and short runs that are far from even (256 rows, all of one of 32
// experts) get narrow tiles that load the weights again and again.
// Token rows of a copy where the runs' lengths are known to the device only: a
// short tile then loads little more than it has.
constexpr int kMxRunBox = 64;

MxPlan mx_gemm_plan(int64_t rows, int64_t N, int experts, int nk, bool runs) {
  const int sms = device_sm_count();
  const auto tiles_of = [&](int tn) {
    const int64_t width = tn > 128 ? 2 * kMxTileN : kMxTileN;
    // runs that can have rows may each end in a tile of their own
    const int64_t more = runs ? (experts < rows ? experts : rows) : (rows % tn != 0);
    return (rows / tn + more) * ((N + width - 1) / width);
  };
  const auto split_of = [&](int tn) {
    int split = 1;
    // no pairs, and a tile for every cluster: the exchange is over when the kernel ends
    if (tn <= 128)
      while (split < 8 && tiles_of(tn) * split * 2 <= sms && nk >= 4 * split) split *= 2;
    return split;
  };
  MxPlan pl{};
  if (runs) {
    const int64_t mean = (rows + experts - 1) / experts;
    pl.tn = mean <= 8 ? 16 : mean <= 24 ? 32 : mean <= 48 ? 64 : 256;
  } else if (rows <= 64) {
    pl.tn = static_cast<int>((rows + 15) / 16 * 16);
  } else {
    int64_t best = INT64_MAX;
    for (int tn = 64; tn <= 256; tn += 16) {
      const int64_t at_once = tn > 128 ? sms / 2 : sms;
      const int split = split_of(tn);
      const int64_t waves = (tiles_of(tn) + at_once - 1) / at_once;
      const int64_t cost = waves * ((nk + split - 1) / split) * (kMxTileN + tn) + (split > 1 ? 800 + 6 * tn : 0);
      if (cost <= best) {
        best = cost;
        pl.tn = tn;
      }
    }
  }
  // wide tiles: a pair of CTAs, each with half of the tokens in shared memory
  pl.pair = pl.tn > 128;
  pl.nt = pl.tn <= 32 ? 32 : pl.tn <= 64 ? 64 : pl.tn <= 128 ? 128 : 256;
  pl.split = split_of(pl.tn);
  const int per = pl.pair ? 2 : pl.split;
  pl.box_rows = pl.pair ? (runs ? kMxRunBox : pl.tn / 2) : pl.tn;
  const int64_t tiles = tiles_of(pl.tn);
  pl.grid = static_cast<int>(tiles < sms / per ? tiles : sms / per) * per;
  return pl;
}

cudaError_t launch_mx_gemm(const CUtensorMap& map_w, const CUtensorMap& map_a, const MxGemmCall& c, const MxPlan& pl,
                           cudaStream_t s) {
  MxGemmArgs p{};
  p.sa = static_cast<const uint8_t*>(c.a_scale);
  p.sw = static_cast<const uint8_t*>(c.b_scale);
  p.off = c.off;
  p.alpha = c.alpha;
  p.out = c.out;
  p.out_ld = c.out_ld;
  p.out_dt = c.out_dt;
  p.E = c.experts;
  p.R = static_cast<int>(c.rows);
  p.N = static_cast<int>(c.N);
  p.nsc = static_cast<int>(c.K / mx_block(c.fmt));
  p.nk = mx_gemm_stages(c.K, c.fmt);
  p.tn = pl.tn;
  p.box = pl.box_rows;
  p.split = pl.split;
  switch (c.fmt) {
    case kFmtNvfp4: return mx_gemm_launch_nt<kFmtNvfp4>(pl, map_w, map_a, p, s);
    case kFmtMxfp4: return mx_gemm_launch_nt<kFmtMxfp4>(pl, map_w, map_a, p, s);
    default: return mx_gemm_launch_nt<kFmtMxfp8>(pl, map_w, map_a, p, s);
  }
}

int mx_gemm_stages(int64_t K, int fmt) {
  const int64_t bytes = fmt == kFmtMxfp8 ? K : K / 2;
  return static_cast<int>((bytes + kMxStageK - 1) / kMxStageK);
}

cudaError_t mx_take_status(unsigned* v) {
  cudaError_t e = cudaMemcpyFromSymbol(v, g_mx_status, 4);
  if (e == cudaSuccess && *v) {
    const unsigned zero = 0;
    e = cudaMemcpyToSymbol(g_mx_status, &zero, 4);
  }
  return e;
}

}  // namespace moe
