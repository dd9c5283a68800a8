// Packed causal grouped-query attention on the 5th-generation tensor cores (tcgen05 + TMEM + TMA).
//
//   o_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = 2^(c q_t . k_j - c max_j),   c = scale log2 e,
// for the tokens t of every request and the keys j <= kv_len - q_len + t of its cache, and, where the
// batch shares a prefix, over all of the prefix's keys as well.
//
// Tile. The G query heads that share a key head are rows of one tile (row = token * G + head), so a
// key block is read once for all of them and one decoding token fills G rows instead of one. A tile
// is two halves of 128 rows (floor(128 / G) tokens each) against key blocks of 128, the page size;
// S = Q K^T and P V run with fp32 accumulators in TMEM: S0 S1 | O0 O1, 128 columns each. The two
// halves are worked in turn, so that the tensor core has one half's products to do while the
// other half is in its softmax; a tile of one half gives its key blocks to both in turn:
//   warp 0      walks the work list, publishes tiles, TMA of Q and of a ring of K / V blocks
//   warp 1      MMA: PV0_j S0_{j+1} PV1_j S1_{j+1}; P is read from TMEM, where it replaces its S
//   warps 4..7  softmax of half 0, warps 8..11 of half 1, one row per thread: running maximum and
//               sum in fp32, P rounded to bf16 (the tensor core's operand type; its error is a
//               relative 2^-8 of each probability, averaged over the keys), O rescaled in TMEM only
//               when the maximum has grown by 2^8 since it was last applied (P <= 2^8, exact at the
//               end because the sum carries the same factor)
// MMAs of one thread complete in order: S_j's commit also means that PV_{j-1} of that half has
// completed, so a softmax warp that has S_j may rescale O, and S_{j+1} may overwrite P_j once PV_j
// was issued.
//
// Work line. All tiles' costs (their visible keys, and a tile's own start and end) are laid
// on one line, the shared prefix's tiles first, then by request, key head and tile; every block
// takes an equal stretch of it, so a stretch may begin and end inside a tile, on a key block. That
// balances prompts of any mix of lengths and splits few long rows over all SMs by the same rule,
// without a host that knows the lengths: a block sums the costs of all requests itself, and
// positions inside a request have a closed form. A tile that lies whole in a stretch is written out
// directly; the others, and all tiles where a prefix is shared (a prefix tile's rows belong to many
// requests), leave O, maximum and sum in fp32 for a second, row-parallel kernel to join. (Joining
// them in the last block to arrive took 13 to 27 us: one SM's loads in flight are too few.)
//
// Keys past a request's end in its last page may hold anything: their scores are replaced, and
// their V rows are zeroed in shared memory, since 0 * NaN would reach the accumulators.
// All waits are bounded; a wait that runs out sets the error word, every role leaves and no row is joined.
//
// What bounds it. Long prompts (four of 3010 to 5001 tokens, 28 heads of 128 over 4, 487 GFLOP): 483 to 498
// us at 1965 MHz (a few calls, 0.98 to 1.01 PFLOP/s), 544 us (0.90) at the 1720 to 1740 MHz that the power
// limit leaves after a second of them. A key block of a half is 3700 clocks from one S to the next: 2000 of softmax
// (exponentials 1280, at the special-function unit's rate; maxima 390; TMEM reads and writes 310), 1024
// of products, the rest hand-offs; the tensor core is busy a little over half of the time. Tried and not
// kept: a quarter or half of the exponentials on the fp32 pipe (equal / 10 % slower), 16 softmax warps
// with a row over four lanes (equal on prompts, 1 us slower on small calls). Answers (96 of 60 to 6000
// keys, 237 MB): 59 to 64 us, 3.7 to 4.0 TB/s; each SM's stretches hold 1 to 10 tiles, and a tile's turnaround (3.6 us:
// last product, output, next tile's first scores) is only partly covered by the loads ahead of it. Small
// calls (10 us): 2 us of work line, 1.5 us of loads, 1.3 us for the first softmax, 1 us of output, and the
// joining kernel.
#include "packed_attention.h"

#include <atomic>
#include <type_traits>

#include "sm100_common.cuh"

namespace appcorr {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kThreads = 384;      // three warpgroups: roles, softmax of half 0, softmax of half 1
constexpr int kMaxBlocks = 256;    // blocks of a launch (one per SM)
constexpr int kTiles = 4;          // published tiles in flight
constexpr int kBlk = 128;          // keys per block = rows per page
// costs on the work line; a key block of two halves (2.0 us) is 128, one of a single half (1.3 us) 80, and a
// tile's own start and end (2.7 us; 3.6 us for a single half; more where 256 rows leave fp32 parts). With one
// price for all key blocks 128 answers after a shared prefix took 71 us for 64, 144 answers of 8 key heads 110
// for 87.
constexpr long kTileCost = 256, kTilePartsCost = 448, kHalfTileCost = 320, kHalfBlockCost = 80;
constexpr long kLeastWork = 128;   // least stretch of a block: at least one block boundary lies in it,
                                   // so the blocks that share a tile's keys are consecutive

template <int DH>
struct Cfg {
  static constexpr int NCH = DH / 64;                       // 64-column chunks
  static constexpr uint32_t CHUNK = 128 * 128;              // one [128 rows x 64] bf16 box
  static constexpr uint32_t TILE = NCH * CHUNK;             // K or V block, or half of Q
  static constexpr int NST = DH == 128 ? 5 : 8;             // ring of K / V blocks
  static constexpr uint32_t SMEM = 2 * TILE + NST * TILE;
  static constexpr uint32_t TAIL = 3072;  // barriers, tiles, scan, row exchange (under 2 KB), and what aligns the base to 1 KB
};

enum : int { kWhole = 1, kEnd = 2, kAlt = 4, kShared = 8 };

// shared-memory descriptors without their address (bits 0..13, address / 16)
constexpr uint64_t sw128_kmajor_desc_base() { return 1ull << 16 | (1024ull >> 4) << 32 | 1ull << 46 | 2ull << 61; }
constexpr uint64_t sw128_mnmajor_desc_base(uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>(lbo >> 4) << 16 | static_cast<uint64_t>(sbo >> 4) << 32 | 1ull << 46 | 2ull << 61;
}

struct Tile {
  int tok0, ntok;  // first packed row and number of tokens
  int lim0;        // last key visible to its first token
  int kv;          // keys of the request
  int hv;          // key head * sub-groups + sub-group
  int jb, n0, n1;  // first key block of this stretch, key blocks of each half
  int flags;       // kWhole: no other block has a part; kAlt: one half's rows, blocks in turn; kShared: prefix
  int slot;        // cut tile: this part's place
  int parts;       // ... and all parts (see pack_parts)
};

// the parts of a cut tile: blocks ca .. cb, of which c0 (where the tile begins) uses its second slot
__device__ __forceinline__ int pack_parts(int c0, int ca, int cb) { return c0 | ca << 8 | cb << 16; }
constexpr int kWholeRow = 255 << 8;  // a row whose tile is whole (no parts: ca > cb)

struct Request {
  int q0, q, past, kv, nt;
  bool shared;  // the prefix: every token of the requests, every key
  bool half;    // the last tile has one half
  long fixed;   // cost of a tile of two halves without its keys
  long base;    // ... and before its own new tokens
  int slope;    // more keys per tile
};

__device__ __forceinline__ Request make_request(const PackedAttnParams& p, int q0, int q1, int kv, bool shared) {
  Request r;
  q0 = max(q0, 0);
  q1 = min(q1, p.N);
  r.q0 = q0;
  r.q = max(q1 - q0, 0);
  r.kv = max(kv, 0);
  r.past = r.kv - r.q;
  r.shared = shared;
  const int tt2 = 2 * p.TT;
  r.nt = (r.q + tt2 - 1) / tt2;
  r.half = r.nt * tt2 - r.q >= p.TT;
  r.fixed = p.row_o != nullptr ? kTilePartsCost : kTileCost;
  r.base = r.fixed + (shared ? r.kv : max(r.past, 0));
  r.slope = shared ? 0 : tt2;
  return r;
}
// entry i of the work line: the prefix (if there is one), then the requests
__device__ __forceinline__ Request load_request(const PackedAttnParams& p, int i) {
  const int b = p.shared_len > 0 ? i - 1 : i;
  if (b < 0) return make_request(p, p.q_start[0], p.q_start[p.B], p.shared_len, true);
  return make_request(p, p.q_start[b], p.q_start[b + 1], p.kv_len[b], false);
}
// the first entry from i on that has new tokens (a whole warp looks, 32 at a time: one after another they
// took 0.2 us each, 3.3 ms for 16384 of them), or E; i lies behind the prefix's entry
__device__ __forceinline__ int next_entry(const PackedAttnParams& p, int i, int E) {
  const int lane = threadIdx.x & 31, b0 = p.shared_len > 0 ? 1 : 0;
  for (; i < E; i += 32) {
    const int b = i + lane - b0;
    const bool some = i + lane < E && min(p.q_start[b + 1], p.N) > max(p.q_start[b], 0);
    const unsigned found = __ballot_sync(0xffffffffu, some);
    if (found) return i + __ffs(found) - 1;
  }
  return E;
}
// cost of the first k tiles of one head
__device__ __forceinline__ long tiles_cost(const Request& r, int k) {
  long c = k * r.base + (long)r.slope * k * (k + 1) / 2;
  if (k == r.nt) {
    if (r.slope) c -= (long)r.nt * r.slope - r.q;
    if (r.half) {  // the last tile's keys at the other price
      const long keys = r.base - r.fixed + (r.slope ? r.q : 0);
      c += kHalfTileCost + keys * kHalfBlockCost / kBlk - r.fixed - keys;
    }
  }
  return c;
}
// key blocks before point w of the line inside the tile [at, at + cost)
__device__ __forceinline__ int cut_block(long w, long at, long cost, int nb, bool half, long fixed) {
  if (w <= at) return 0;
  if (w >= at + cost) return nb;
  const long s = half ? (w - at - kHalfTileCost + kHalfBlockCost / 2) / kHalfBlockCost : (w - at - fixed + kBlk / 2) / kBlk;
  return static_cast<int>(min(max(s, 0L), static_cast<long>(nb)));
}

// Programmatic dependent launch: a kernel of this file starts while the one before it ends, and waits
// here before it touches what that one (or any before it) wrote.
__device__ __forceinline__ void wait_for_earlier_kernels() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_later_kernels_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Bounded wait of a whole warp. It counts polls and reads no clock: the waits lie on the chain of S,
// softmax and P V, and the clock's code beside them cost 2 to 4 %. The hardware suspends a poll that
// fails for 1.3 us, so 2^20 of them are 1.4 s; tiles take less than a few milliseconds.
__device__ __forceinline__ bool poll(uint32_t bar, uint32_t parity, int* err, int code) {
#pragma unroll 1
  for (int i = 0; i < (1 << 20); ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255) == 255 && error_raised(err)) return false;
  }
  record_error(err, code);
  return false;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, poll(bar, parity, err, code));
}
// two barriers at once: one latency where both are done
__device__ __forceinline__ bool warp_wait2(uint32_t bar0, uint32_t parity0, uint32_t bar1, uint32_t parity1, int* err, int code) {
  const bool d0 = mbar_try_wait(bar0, parity0), d1 = mbar_try_wait(bar1, parity1);
  if (__all_sync(0xffffffffu, d0 && d1)) return true;
  return warp_wait(bar0, parity0, err, code) && warp_wait(bar1, parity1, err, code);
}

// MMA and commit by one elected lane of a warp whose control flow is uniform. The election sits
// inside the instruction's own predicate: under an `if (lane == 0)` the operands of every MMA are moved
// to uniform registers one by one and the issue of 8 MMAs (512 clocks of work) takes 460 clocks, this
// way 310, so that the tensor core's queue stays ahead of the waits in between.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar)
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// two floats of one 64-bit register pair at a time
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 16 TMEM lanes x 64 columns: register 4 g + e of a thread holds row lane / 4 (+ 8 for e >= 2) and
// column 8 g + 2 (lane % 4) + (e & 1)
__device__ __forceinline__ void tmem_ld_16x64(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// 4 x 4 transposition inside a quad of lanes: register i of lane q becomes register q of lane i
__device__ __forceinline__ void quad_transpose(uint32_t (&r)[4], int q) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint32_t w = __shfl_xor_sync(0xffffffffu, q & 1 ? r[i] : r[i + 1], 1);
    if (q & 1) r[i] = w;
    else r[i + 1] = w;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t w = __shfl_xor_sync(0xffffffffu, q & 2 ? r[i] : r[i + 2], 2);
    if (q & 2) r[i] = w;
    else r[i + 2] = w;
  }
}

template <int DH>
__global__ void __launch_bounds__(kThreads, 1)
    packed_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmQ1,
                            const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ PackedAttnParams p) {
  using C = Cfg<DH>;
  constexpr int NST = C::NST, NCH = C::NCH;
  constexpr uint32_t IDESC_S = idesc_bf16_f32(128, kBlk);
  constexpr uint32_t IDESC_O = idesc_bf16_f32_b(128, DH, true);
  constexpr uint32_t O_COL = 256;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + 2 * C::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::SMEM);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 1;
  uint64_t* s_full = bars + 2;            // 2
  uint64_t* p_full = bars + 4;            // 2
  uint64_t* o_full = bars + 6;            // 2
  uint64_t* o_empty = bars + 8;           // 2
  uint64_t* x_full = bars + 10;           // 4: half 1's maxima and sums of a kAlt tile, per 32 rows
  uint64_t* x_empty = bars + 14;          // 4
  uint64_t* t_full = bars + 18;           // kTiles
  uint64_t* t_empty = t_full + kTiles;    // kTiles
  uint64_t* done = t_empty + kTiles;
  uint64_t* full = done + 1;              // NST
  uint64_t* empty = full + NST;           // NST (43 barriers at the most)
  float2* s_ml = reinterpret_cast<float2*>(bars + 44);    // [128]
  Tile* tiles = reinterpret_cast<Tile*>(s_ml + 128);
  long* scan = reinterpret_cast<long*>(tiles + kTiles);   // the warps' sums, the begin's offset
  int* s_int = reinterpret_cast<int*>(scan + kThreads / 32 + 1);  // begin's entry, TMEM base, the entry's tokens and keys
  static_assert(sizeof(Tile) * kTiles % 8 == 0 && 44 * 8 + 1024 + sizeof(Tile) * kTiles + 8 * (kThreads / 32 + 1) + 24 <= 2048,
                "the tail holds what lies in it");

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int me = blockIdx.x;

  if (warp == 0 && lane == 0) {
    mbar_init(smem_addr(q_full), 1);
    mbar_init(smem_addr(q_empty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&s_full[i]), 1);
      mbar_init(smem_addr(&p_full[i]), 4);
      mbar_init(smem_addr(&o_full[i]), 1);
      mbar_init(smem_addr(&o_empty[i]), 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_addr(&x_full[i]), 1);
      mbar_init(smem_addr(&x_empty[i]), 1);
    }
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(smem_addr(&t_full[i]), 1);
      mbar_init(smem_addr(&t_empty[i]), 9);
    }
    mbar_init(smem_addr(done), 1);
    for (int i = 0; i < NST; ++i) {
      mbar_init(smem_addr(&full[i]), 1);
      mbar_init(smem_addr(&empty[i]), 1);
    }
    fence_barrier_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(smem_addr(&s_int[1]), 512);
    tmem_relinquish();
  }

  wait_for_earlier_kernels();
  let_later_kernels_start();

  // ---------------------------------------------------------------- this block's stretch of the line
  const int E = p.B + (p.shared_len > 0);
  long W = 0;  // the line's length: with few entries the scan below finds it, with many a sum before it
  if (E > kThreads) {
    long sum = 0;
    for (int i = tid; i < E; i += kThreads) {
      const Request r = load_request(p, i);
      sum += p.Hv * tiles_cost(r, r.nt);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) scan[warp] = sum;
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) W += scan[w];
  }
  long L = 0, w0 = 0, w1 = 0, base = 0;  // stretches are L long, block c's begins at c * L
  for (int i0 = 0; i0 < E; i0 += kThreads) {
    if (i0 || E > kThreads) __syncthreads();
    const int i = i0 + tid;
    long v = 0;
    Request r{};
    if (i < E) {
      r = load_request(p, i);
      v = p.Hv * tiles_cost(r, r.nt);
    }
    long inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long up = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += up;
    }
    if (lane == 31) scan[warp] = inc;
    __syncthreads();
    long before = base, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      const long s = scan[w];
      if (w < warp) before += s;
      all += s;
    }
    if (i0 == 0) {
      if (E <= kThreads) W = all;
      L = max((W + gridDim.x - 1) / static_cast<long>(gridDim.x), kLeastWork);
      w0 = me * L;
      w1 = min(w0 + L, W);
    }
    if (before + inc - v <= w0 && w0 < before + inc) {
      s_int[0] = i;
      s_int[2] = r.q0;
      s_int[3] = r.q0 + r.q;
      s_int[4] = r.kv;
      scan[kThreads / 32] = w0 - (before + inc - v);
    }
    base += all;
    if (base > w0) break;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_int[1];
  if (w0 >= W) {
    if (tid == 0) p.cuts[me].parts = -1;
    if (warp == 1) tmem_dealloc(tmem, 512);
    return;
  }

  // registers: 384 threads start with 168 each (64512); the roles keep 88, the softmax threads get
  // 208 (128 x (88 + 208 + 208) = 64512)
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0) {
      // ---------------------------------------------------------------------------- work list + TMA
      bool ok = true;
      int e = s_int[0];
      Request r = make_request(p, s_int[2], s_int[3], s_int[4], p.shared_len > 0 && e == 0);
      const long head_cost = tiles_cost(r, r.nt);
      const long off = scan[kThreads / 32];
      int hv = static_cast<int>(off / head_cost), t = 0;
      long at = w0;
      {  // the tile of that head that holds the begin
        const long rem = off - hv * head_cost;
        int lo = 0, hi = r.nt;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (tiles_cost(r, mid) <= rem) lo = mid;
          else hi = mid;
        }
        t = lo;
        at = w0 - (rem - tiles_cost(r, lo));
      }
      const int tt2 = 2 * p.TT;
      uint32_t it = 0;  // K / V blocks issued
      int nq = 0, np = 0, cut_parts = -1, cut_tok0 = 0, cut_ntok = 0, cut_hv = 0;
      while (ok && at < w1) {
        const long cost = tiles_cost(r, t + 1) - tiles_cost(r, t);
        const int t0 = t * tt2, ntok = min(tt2, r.q - t0);
        const int vis1 = r.shared ? r.kv : min(max(r.past + t0 + ntok, 0), r.kv);
        const int vis0 = r.shared ? r.kv : min(max(r.past + t0 + min(ntok, p.TT), 0), r.kv);
        const int nb = vis1 / kBlk + (vis1 % kBlk != 0), nb0 = vis0 / kBlk + (vis0 % kBlk != 0);
        const bool owner = at >= w0;
        const int jb = cut_block(w0, at, cost, nb, ntok <= p.TT, r.fixed), je = cut_block(w1, at, cost, nb, ntok <= p.TT, r.fixed);
        const bool whole = jb == 0 && je == nb;
        const int kvh = hv / p.ng, b = p.shared_len > 0 ? e - 1 : e;
        const int* pages = r.shared ? p.prefix : p.table != nullptr ? p.table + b * p.ld_table : nullptr;
        const int npages = r.shared ? p.prefix_pages : p.W;
        auto fetch_pages = [&](int j) { return jb + j + lane < npages && j + lane < je - jb ? pages[jb + j + lane] : -1; };
        int pg = pages != nullptr ? fetch_pages(0) : 0;  // on its way while the parts are worked out
        int parts = 0;
        if (!whole && (je > jb || owner)) {  // the blocks that share this tile: their stretches meet [at, at + cost)
          const int c0 = static_cast<int>(at / L), c1 = static_cast<int>((at + cost - 1) / L);
          int ca = -1, cb = -1;
#pragma unroll 1
          for (int c = c0; c <= c1; c += 32) {
            const int cl = c + lane;
            const unsigned some = __ballot_sync(0xffffffffu, cl <= c1 && cut_block((cl + 1) * L, at, cost, nb, ntok <= p.TT, r.fixed) >
                                                                             cut_block(cl * L, at, cost, nb, ntok <= p.TT, r.fixed));
            if (some) {
              if (ca < 0) ca = c + __ffs(some) - 1;
              cb = c + 31 - __clz(some);
            }
          }
          parts = pack_parts(c0, ca, cb);
          if (owner && cb > ca) {
            cut_parts = parts;
            cut_tok0 = r.q0 + t0;
            cut_ntok = ntok;
            cut_hv = hv;
          }
        }
        if (je > jb || (nb == 0 && owner)) {
          const bool alt = ntok <= p.TT && je - jb > 1;
          ok = warp_wait(smem_addr(&t_empty[np % kTiles]), ((np / kTiles) & 1) ^ 1, p.err, kErrTimeoutProducer);
          if (!ok) break;
          if (lane == 0) {
            Tile& out = tiles[np % kTiles];
            out.tok0 = r.q0 + t0;
            out.ntok = ntok;
            out.lim0 = r.past + t0;
            out.kv = r.kv;
            out.hv = hv;
            out.jb = jb;
            out.n0 = alt ? (je - jb + 1) / 2 : min(max(nb0 - jb, 0), je - jb);
            out.n1 = alt ? (je - jb) / 2 : (ntok > p.TT ? je - jb : 0);
            out.flags = (whole ? kWhole : 0) | (alt ? kAlt : 0) | (r.shared ? kShared : 0);
            out.slot = 2 * me + owner;
            out.parts = parts;
            mbar_arrive(smem_addr(&t_full[np % kTiles]));
          }
          ++np;
          for (int j = 0; ok && j < je - jb; ++j) {
            const int blk = jb + j;
            int row;
            if (pages != nullptr) {
              if ((j & 31) == 0) {
                if (j) pg = fetch_pages(j);
                if (pg < 0 || pg >= p.pages) pg = p.pages;  // no page: past the pool, where TMA fills zeros
              }
              row = __shfl_sync(0xffffffffu, pg, j & 31) * kBlk;
            } else {
              const int k0 = p.k_start[b];
              row = k0 >= 0 && blk <= (p.key_rows - k0) / kBlk ? k0 + blk * kBlk : p.key_rows;
            }
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
              const uint32_t st = it % NST;
              ok = ok && warp_wait(smem_addr(&empty[st]), ((it / NST) & 1) ^ 1, p.err, kErrTimeoutProducer);
              if (!ok) break;
              if (lane == 0) {
                const uint32_t fb = smem_addr(&full[st]);
                mbar_arrive_expect_tx(fb, C::TILE);
                for (int c = 0; c < NCH; ++c)
                  tma_load_2d(smem_addr(sKV + st * C::TILE + c * C::CHUNK), kv ? &tmV : &tmK, fb, kvh * DH + c * 64, row);
              }
              ++it;
              if (kv == 0 && j == 0) {  // Q behind the first K block: its buffer frees up last
                ok = warp_wait(smem_addr(q_empty), (nq & 1) ^ 1, p.err, kErrTimeoutProducer);
                if (!ok) break;
                if (lane == 0) {
                  const uint32_t qb = smem_addr(q_full);
                  const bool one = ntok == 1;  // a single token: its G rows alone
                  const int halves = ntok > p.TT ? 2 : 1;
                  const uint32_t bytes = 128u * p.G * (one ? 1 : p.TT);
                  mbar_arrive_expect_tx(qb, bytes * NCH * halves);
                  for (int hf = 0; hf < halves; ++hf)
                    for (int c = 0; c < NCH; ++c)
                      tma_load_3d(smem_addr(sQ + hf * C::TILE + c * C::CHUNK), one ? &tmQ1 : &tmQ, qb, c * 64, hv * p.G,
                                  r.q0 + t0 + hf * p.TT);
                }
                ++nq;
              }
            }
          }
        }
        at += cost;
        if (++t == r.nt) {
          t = 0;
          if (++hv == p.Hv) {
            hv = 0;
            if (at >= w1) break;  // before looking further: what follows may be thousands of idle requests
            e = next_entry(p, e + 1, E);
            if (e >= E) break;
            r = load_request(p, e);
          }
        }
      }
      ok = ok && warp_wait(smem_addr(&t_empty[np % kTiles]), ((np / kTiles) & 1) ^ 1, p.err, kErrTimeoutProducer);
      if (lane == 0) {
        if (ok) {
          tiles[np % kTiles].flags = kEnd;
          mbar_arrive(smem_addr(&t_full[np % kTiles]));
        }
        CutTile& cut = p.cuts[me];
        cut.parts = cut_parts;
        cut.tok0 = cut_tok0;
        cut.ntok = cut_ntok;
        cut.hv = cut_hv;
      }
      if (!ok) {  // let the copies in flight land before the block ends
        const uint32_t from = it > NST ? it - NST : 0;
        for (uint32_t i = from; i < it; ++i) mbar_wait(smem_addr(&full[i % NST]), (i / NST) & 1, nullptr, 0);
        if (nq) mbar_wait(smem_addr(q_full), (nq - 1) & 1, nullptr, 0);
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------------------------- MMA
      bool ok = true;
      uint32_t it = 0;
      int nq = 0;
      int np_[2] = {0, 0}, no_[2] = {0, 0};  // P tiles and O tiles consumed per half
      const uint32_t qa = smem_addr(sQ), kva = smem_addr(sKV);
      auto landed = [&](uint32_t i) { return warp_wait(smem_addr(&full[i % NST]), (i / NST) & 1, p.err, kErrTimeoutMma); };
      constexpr uint64_t kDescK = sw128_kmajor_desc_base(), kDescV = sw128_mnmajor_desc_base(C::CHUNK, 1024);
      auto issue_s = [&](int hf, int qh, uint32_t i) {  // S of half hf from Q half qh and ring entry i
        const uint64_t ka = kDescK | ((kva + (i % NST) * C::TILE) >> 4), qb = kDescK | ((qa + qh * C::TILE) >> 4);
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
          const uint32_t off = ((k >> 2) * C::CHUNK + (k & 3) * 32) >> 4;
          mma_ss(tmem + hf * 128, qb + off, ka + off, IDESC_S, k > 0);
        }
        mma_commit(smem_addr(&s_full[hf]));
      };
      // V rows of keys that do not exist become zeros; `live` of the 128 exist
      auto clear_dead = [&](uint32_t i, int live) {
        if (live >= kBlk) return;
        for (int x = lane; x < (kBlk - live) * 8; x += 32)
#pragma unroll
          for (int c = 0; c < NCH; ++c)
            *reinterpret_cast<uint4*>(sKV + (i % NST) * C::TILE + c * C::CHUNK + live * 128 + x * 16) = make_uint4(0, 0, 0, 0);
        fence_proxy_async_smem();
        __syncwarp();
      };
      auto issue_pv = [&](int hf, uint32_t i, bool first, bool last) -> bool {
        if (!warp_wait(smem_addr(&p_full[hf]), np_[hf] & 1, p.err, kErrTimeoutMma)) return false;
        ++np_[hf];
        if (first) {
          if (!warp_wait(smem_addr(&o_empty[hf]), (no_[hf] & 1) ^ 1, p.err, kErrTimeoutMma)) return false;
          ++no_[hf];
        }
        tc_fence_after();
        const uint64_t va = kDescV | ((kva + (i % NST) * C::TILE) >> 4);
#pragma unroll
        for (int k = 0; k < kBlk / 16; ++k)
          mma_ts(tmem + O_COL + hf * 128, tmem + hf * 128 + k * 8, va + k * (2048 >> 4), IDESC_O, (!first || k > 0) ? 1u : 0u);
        if (last) mma_commit(smem_addr(&o_full[hf]));
        return true;
      };
      for (int np = 0;; ++np) {
        ok = warp_wait(smem_addr(&t_full[np % kTiles]), (np / kTiles) & 1, p.err, kErrTimeoutMma);
        if (!ok) break;
        const Tile& tl = tiles[np % kTiles];
        // broadcast, so that the compiler keeps the loops below uniform
        const int flags = __shfl_sync(0xffffffffu, tl.flags, 0), n0 = __shfl_sync(0xffffffffu, tl.n0, 0),
                  n1 = __shfl_sync(0xffffffffu, tl.n1, 0), kv = __shfl_sync(0xffffffffu, tl.kv, 0),
                  jb = __shfl_sync(0xffffffffu, tl.jb, 0);
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&t_empty[np % kTiles]));
        if (flags & kEnd) break;
        const int cnt = flags & kAlt ? n0 + n1 : max(n0, n1);
        if (cnt == 0) continue;
        ok = landed(it) && warp_wait(smem_addr(q_full), nq & 1, p.err, kErrTimeoutMma);
        if (!ok) break;
        ++nq;
        tc_fence_after();
        if (flags & kAlt) {
          // block j in half j & 1: S_0 S_1, then PV_j S_{j+2}; ring entries 2j (K), 2j + 1 (V)
          const uint32_t i0 = it;
          issue_s(0, 0, i0);
          mma_commit(smem_addr(&empty[i0 % NST]));
          ok = landed(i0 + 2);
          if (!ok) break;
          tc_fence_after();
          issue_s(1, 0, i0 + 2);
          mma_commit(smem_addr(&empty[(i0 + 2) % NST]));
          if (cnt == 2) mma_commit(smem_addr(q_empty));
          for (int j = 0; ok && j < cnt; ++j) {
            const uint32_t iv = i0 + 2 * j + 1, ik = iv + 3;
            ok = landed(iv);
            if (!ok) break;
            clear_dead(iv, kv - (jb + j) * kBlk);
            ok = issue_pv(j & 1, iv, j < 2, j + 2 >= cnt);
            if (!ok) break;
            mma_commit(smem_addr(&empty[iv % NST]));
            if (j + 2 < cnt) {
              ok = landed(ik);
              if (!ok) break;
              tc_fence_after();
              issue_s(j & 1, 0, ik);
              mma_commit(smem_addr(&empty[ik % NST]));
              if (j + 3 == cnt) mma_commit(smem_addr(q_empty));
            }
          }
          it = i0 + 2 * cnt;
        } else {
          if (n0 > 0) issue_s(0, 0, it);
          if (n1 > 0) issue_s(1, 1, it);
          mma_commit(smem_addr(&empty[it % NST]));
          if (cnt == 1) mma_commit(smem_addr(q_empty));
          ++it;
          for (int j = 0; ok && j < cnt; ++j) {
            const uint32_t iv = it, ik = it + 1;
            const bool more = j + 1 < cnt;
            ok = more ? warp_wait2(smem_addr(&full[iv % NST]), (iv / NST) & 1, smem_addr(&full[ik % NST]), (ik / NST) & 1, p.err, kErrTimeoutMma)
                      : landed(iv);
            if (!ok) break;
            clear_dead(iv, kv - (jb + j) * kBlk);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int nh = hf ? n1 : n0;
              if (j >= nh) continue;
              ok = issue_pv(hf, iv, j == 0, j + 1 == nh);
              if (!ok) break;
              if (j + 1 < nh) issue_s(hf, hf, ik);
            }
            if (!ok) break;
            mma_commit(smem_addr(&empty[iv % NST]));
            if (more) {
              mma_commit(smem_addr(&empty[ik % NST]));
              if (j + 2 == cnt) mma_commit(smem_addr(q_empty));
            }
            it += more ? 2 : 1;
          }
        }
        if (!ok) break;
      }
      if (!ok) {  // products in flight end before TMEM is given back
        mma_commit(smem_addr(done));
        mbar_wait(smem_addr(done), 0, nullptr, 0);
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    // ------------------------------------------------------------------------------ softmax + output
    const int qd = warp & 3, hf = (warp - 4) >> 2;
    const int row = qd * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(qd * 32) << 16;
    const uint32_t s_addr = tmem + lane_base + hf * 128, o_addr = tmem + lane_base + O_COL + hf * 128;
    const int rtok = row / p.G, rhead = row - rtok * p.G;  // this row's token and head inside the half
    const float sl2 = p.scale_log2;
    int ns = 0, no = 0, no1 = 0, nx = 0;
    bool ok = true;
    for (int np = 0;; ++np) {
      ok = warp_wait(smem_addr(&t_full[np % kTiles]), (np / kTiles) & 1, p.err, kErrTimeoutEpilogue);
      if (!ok) break;
      const Tile& tl = tiles[np % kTiles];
      const int flags = tl.flags;
      if (flags & kEnd) break;
      auto release = [&] {  // this warp no longer reads the tile's description
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&t_empty[np % kTiles]));
      };
      const bool alt = flags & kAlt;
      const int cnt = hf ? tl.n1 : tl.n0, step = alt ? 2 : 1;
      const int tk = (alt ? 0 : hf * p.TT) + rtok;
      const bool valid = rtok < p.TT && tk < tl.ntok;
      const bool alive = __any_sync(0xffffffffu, valid);  // some row of this warp is stored
      const int klim = flags & kShared ? tl.kv - 1 : min(tl.kv - 1, tl.lim0 + tk);
      const int over0 = klim - (tl.jb + (alt ? hf : 0)) * kBlk;  // last visible key, from the first block's start
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = 0; j < cnt; ++j, ++ns) {
        ok = warp_wait(smem_addr(&s_full[hf]), ns & 1, p.err, kErrTimeoutEpilogue);
        if (!ok) break;
        tc_fence_after();
        if (alive) {
          float sv[kBlk];
          {
            uint32_t* u = reinterpret_cast<uint32_t*>(sv);
#pragma unroll
            for (int c = 0; c < kBlk / 32; ++c) tmem_ld32(s_addr + c * 32, *reinterpret_cast<uint32_t(*)[32]>(u + c * 32));
            tmem_wait_ld();
          }
          const int over = over0 - j * step * kBlk;  // last visible key of this block
          if (__any_sync(0xffffffffu, over < kBlk - 1)) {
#pragma unroll
            for (int i = 0; i < kBlk; ++i) sv[i] = i <= over ? sv[i] : -INFINITY;
          }
          float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
          for (int i = 4; i < kBlk; i += 8) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
              if (i + 2 * u + 1 < kBlk) mx[u] = max3(mx[u], sv[i + 2 * u], sv[i + 2 * u + 1]);
          }
          const float top = max3(fmaxf(mx[0], mx[1]), mx[2], mx[3]);
          const bool grow = valid && (top - m_run) * sl2 > 8.f;
          float corr = 1.f;
          if (grow) {
            corr = ex2_approx((m_run - top) * sl2);
            m_run = top;
            l_run *= corr;
          }
          if (j > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
            for (int c = 0; c < DH / 32; ++c) {
              uint32_t u[32];
              tmem_ld32(o_addr + c * 32, u);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) u[i] = __float_as_uint(__uint_as_float(u[i]) * corr);
              tmem_st32(o_addr + c * 32, u);
            }
          }
          const float moff = m_run == -INFINITY ? 0.f : m_run * sl2;
          const uint64_t sl2x2 = pack2(sl2, sl2), offx2 = pack2(-moff, -moff);
          uint64_t ls[2] = {0, 0};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              float e0, e1;
              unpack2(fma2(pack2(sv[c * 64 + 2 * i], sv[c * 64 + 2 * i + 1]), sl2x2, offx2), e0, e1);
              e0 = ex2_approx(e0);
              e1 = ex2_approx(e1);
              ls[i & 1] = add2(ls[i & 1], pack2(e0, e1));
              pk[i] = pack_bf16x2(e0, e1);
            }
            tmem_st32(s_addr + c * 32, pk);
          }
          float l0, l1;
          unpack2(add2(ls[0], ls[1]), l0, l1);
          l_run += l0 + l1;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&p_full[hf]));
      }
      if (!ok) break;
      float mlog = m_run == -INFINITY ? -INFINITY : m_run * sl2;  // maximum in log2 units
      if (alt && hf == 1) {  // half 0's warp of the same rows reads this half's O and writes the result
        if (alive) {
          ok = warp_wait(smem_addr(&x_empty[qd]), (nx & 1) ^ 1, p.err, kErrTimeoutEpilogue);
          if (!ok) break;
          ++nx;
          s_ml[row] = make_float2(mlog, l_run);
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&x_full[qd]));
        }
        ok = warp_wait(smem_addr(&o_full[1]), no & 1, p.err, kErrTimeoutEpilogue);  // keeps this warp's phase count in step
        if (!ok) break;
        ++no;
        release();
        continue;
      }
      if (cnt > 0) {
        ok = warp_wait(smem_addr(&o_full[hf]), no & 1, p.err, kErrTimeoutEpilogue);
        if (!ok) break;
        ++no;
      }
      float a0 = 1.f, a1 = 0.f;
      if (hf == 0 && (alt || tl.n1 > 0)) {
        if (alt) {
          ok = warp_wait(smem_addr(&o_full[1]), no1 & 1, p.err, kErrTimeoutEpilogue);
          if (!ok) break;
          if (alive) {
            ok = warp_wait(smem_addr(&x_full[qd]), nx & 1, p.err, kErrTimeoutEpilogue);
            if (!ok) break;
            ++nx;
            const float2 ml = s_ml[row];
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_addr(&x_empty[qd]));
            const float top = fmaxf(mlog, ml.x), safe = top == -INFINITY ? 0.f : top;
            a0 = ex2_approx(mlog - safe);
            a1 = ex2_approx(ml.x - safe);
            l_run = a0 * l_run + a1 * ml.y;
            mlog = top;
          }
        }
        ++no1;
      }
      tc_fence_after();
      auto o_done = [&] {  // the accumulators may be overwritten
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (cnt > 0) mbar_arrive(smem_addr(&o_empty[hf]));
          if (alt) mbar_arrive(smem_addr(&o_empty[1]));
        }
      };
      if (!alive) {
        o_done();
        release();
        continue;
      }
      const long tok = tl.tok0 + tk;
      const int head = tl.hv * p.G + rhead;
      const long orow = tok * p.H + head;
      // O goes out 16 rows x 64 columns at a time, in an order in which a quad of lanes holds 64 bytes of
      // a row (with a row per lane every store touches 32 rows). The loops stay rolled: this code runs
      // once per tile, and unrolled it spent 4000 clocks and more on fetching instructions.
      const int q4 = lane & 3;
      auto load_o = [&](int h, int c, uint32_t (&x)[32]) {  // rows 16 h .. 16 h + 15, columns 64 c .. 64 c + 63
        __syncwarp();
        if (cnt > 0) {
          tmem_ld_16x64(o_addr + (h << 20) + c * 64, x);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = 0u;
        }
        if (alt) {  // and half 1's accumulators of the same rows
          uint32_t u[32];
          tmem_ld_16x64(o_addr + 128 + (h << 20) + c * 64, u);
          const int r0 = 16 * h + lane / 4;
          const float f0 = __shfl_sync(0xffffffffu, a0, r0), f1 = __shfl_sync(0xffffffffu, a1, r0);
          const float g0 = __shfl_sync(0xffffffffu, a0, r0 + 8), g1 = __shfl_sync(0xffffffffu, a1, r0 + 8);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            x[i] = __float_as_uint(__uint_as_float(x[i]) * (i & 2 ? g0 : f0) + __uint_as_float(u[i]) * (i & 2 ? g1 : f1));
        }
      };
      const unsigned stored = __ballot_sync(0xffffffffu, valid);
      if ((flags & kWhole) && p.row_o == nullptr) {  // the tile's only part: the result
        const float inv = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f;
        const long at = tok * p.ldo + (long)head * DH;
#pragma unroll 1
        for (int hc = 0; hc < DH / 32; ++hc) {
          const int h = hc & 1, c = hc >> 1;
          if (!((stored >> (16 * h)) & 0xFFFFu)) continue;
          uint32_t x[32];
          load_o(h, c, x);
#pragma unroll
          for (int k = 0; k < 2; ++k) {  // rows lane / 4 and lane / 4 + 8 of the 16
            if (!((stored >> (16 * h + 8 * k)) & 0xFFu)) continue;
            const int r = 16 * h + 8 * k + lane / 4;
            const float w = __shfl_sync(0xffffffffu, inv, r);
            bf16* dst = p.o + __shfl_sync(0xffffffffu, at, r) + c * 64 + q4 * 8;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
              uint32_t v[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int e = (4 * b + i) * 4 + k * 2;
                v[i] = pack_bf16x2(__uint_as_float(x[e]) * w, __uint_as_float(x[e + 1]) * w);
              }
              quad_transpose(v, q4);
              if ((stored >> r) & 1) *reinterpret_cast<uint4*>(dst + b * 32) = make_uint4(v[0], v[1], v[2], v[3]);
            }
          }
        }
        o_done();
        if (valid && p.lse != nullptr) p.lse[orow] = (mlog + log2f(l_run)) * 0.69314718055994531f;
      } else {  // a part: O, maximum and sum for the joining kernel
        const long cls = flags & kShared ? (long)p.N * p.H : 0;
        const long prow = flags & kWhole ? cls + orow : (long)tl.slot * kPaRows + (alt ? 0 : hf * 128) + row;
        float* part_o = flags & kWhole ? p.row_o : p.slots;
        float* part_ml = flags & kWhole ? p.row_ml : p.slot_ml;
#pragma unroll 1
        for (int hc = 0; hc < DH / 32; ++hc) {
          const int h = hc & 1, c = hc >> 1;
          if (!((stored >> (16 * h)) & 0xFFFFu)) continue;
          uint32_t x[32];
          load_o(h, c, x);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (!((stored >> (16 * h + 8 * k)) & 0xFFu)) continue;
            const int r = 16 * h + 8 * k + lane / 4;
            float* dst = part_o + __shfl_sync(0xffffffffu, prow, r) * DH + c * 64 + (q4 & 1) * 8 + (q4 & 2) * 2;
#pragma unroll
            for (int b = 0; b < 4; ++b) {  // two 8-column groups: even lanes take the first, odd ones the second
              const int e = 2 * b * 4 + k * 2;
              uint32_t v[2][2] = {{x[e], x[e + 1]}, {x[e + 4], x[e + 5]}};
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const uint32_t w = __shfl_xor_sync(0xffffffffu, lane & 1 ? v[0][i] : v[1][i], 1);
                if (lane & 1) v[0][i] = w;
                else v[1][i] = w;
              }
              if ((stored >> r) & 1) *reinterpret_cast<uint4*>(dst + b * 16) = make_uint4(v[0][0], v[0][1], v[1][0], v[1][1]);
            }
          }
        }
        o_done();
        if (valid) {
          *reinterpret_cast<float2*>(part_ml + prow * 2) = make_float2(mlog, l_run);
          // with the row's place inside the tile, where the slots have it
          if (p.row_o != nullptr) p.row_parts[cls + orow] = flags & kWhole ? kWholeRow : tl.parts | ((alt ? 0 : hf * 128) + row) << 24;
        }
      }
      release();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ------------------------------------------------------------------------------------ joining parts
// One row by one warp: part i (of `count`) has its maximum and sum at ml(i), its O at o(i); a lane
// holds D / 32 columns. What it costs is reads after one another (about a microsecond each, for lines
// that other SMs have just written): the lanes read up to 32 parts' maxima at once, and the O rows of
// the first FLY parts are in flight together with them.
template <int DH, int FLY, typename Ml, typename O>
__device__ __forceinline__ void join_row(int count, Ml ml_of, O o_of, __nv_bfloat16* out, float* lse) {
  constexpr int CPL = DH / 32;
  using Vec = typename std::conditional<CPL == 4, float4, float2>::type;
  const int lane = threadIdx.x & 31;
  float top = -INFINITY, total = 0.f, acc[CPL];
#pragma unroll
  for (int k = 0; k < CPL; ++k) acc[k] = 0.f;
#pragma unroll 1
  for (int i0 = 0; i0 < count; i0 += 32) {
    const int m = min(32, count - i0);
    Vec f[FLY];
    auto fetch = [&](int i) {
#pragma unroll
      for (int u = 0; u < FLY; ++u)
        if (i + u < m) f[u] = *reinterpret_cast<const Vec*>(o_of(i0 + i + u) + lane * CPL);
    };
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < m) ml = *reinterpret_cast<const float2*>(ml_of(i0 + lane));
    fetch(0);
    float t = ml.x;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
    t = fmaxf(t, top);
    const float safe = t == -INFINITY ? 0.f : t;
    const float old = ex2_approx(top - safe), w = ex2_approx(ml.x - safe);
    float sum = w * ml.y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    total = total * old + sum;
    top = t;
#pragma unroll
    for (int k = 0; k < CPL; ++k) acc[k] *= old;
#pragma unroll 1
    for (int i = 0; i < m; i += FLY) {
      if (i) fetch(i);
#pragma unroll
      for (int u = 0; u < FLY; ++u) {
        const float ws = __shfl_sync(0xffffffffu, w, (i + u) & 31);
        if (i + u < m) {
          acc[0] = fmaf(ws, f[u].x, acc[0]);
          acc[1] = fmaf(ws, f[u].y, acc[1]);
          if constexpr (CPL == 4) {
            acc[2] = fmaf(ws, f[u].z, acc[2]);
            acc[3] = fmaf(ws, f[u].w, acc[3]);
          }
        }
      }
    }
  }
  const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
  if constexpr (CPL == 4)
    *reinterpret_cast<uint2*>(out + lane * CPL) =
        make_uint2(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(out + lane * CPL) = pack_bf16x2(acc[0] * inv, acc[1] * inv);
  if (lse != nullptr && lane == 0) *lse = (top + log2f(total)) * 0.69314718055994531f;
}

// place of part i: inside the slots whatever the part numbers are (after a wait that ran out they may be
// what the workspace held before)
__device__ __forceinline__ long part_row(int parts, int i, int row, int blocks) {
  const int c0 = parts & 255, c = min(((parts >> 8) & 255) + i, blocks - 1);
  return (long)(2 * c + (c == c0)) * kPaRows + row;
}
__device__ __forceinline__ int part_count(int parts) { return ((parts >> 16) & 255) - ((parts >> 8) & 255) + 1; }

constexpr int kJoinThreads = 256;
constexpr int kCutBlocksPerSm = 4;  // 64 registers: the first four parts stay in flight without spills

// The rows of all cut tiles (at most one begins in each block of the attention kernel), shared out evenly.
template <int DH>
__global__ void __launch_bounds__(kJoinThreads, kCutBlocksPerSm) join_cut_tiles_kernel(PackedAttnParams p, int blocks) {
  static_assert(kMaxBlocks <= kJoinThreads, "one thread per noted tile");
  __shared__ CutTile s_cut[kMaxBlocks];
  __shared__ int s_end[kMaxBlocks];  // rows up to and with this tile's
  __shared__ int s_warp[kMaxBlocks / 32];
  wait_for_earlier_kernels();
  let_later_kernels_start();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int rows = 0;
  if (tid < kMaxBlocks) {
    CutTile cut;
    cut.parts = -1;
    const int failed = *p.err;  // the parts are not there: no row is joined
    if (tid < blocks) cut = p.cuts[tid];
    if (failed != 0) cut.parts = -1;
    s_cut[tid] = cut;
    rows = cut.parts >= 0 ? cut.ntok * p.G : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, rows, o);
      if (lane >= o) rows += up;
    }
    if (lane == 31) s_warp[warp] = rows;
  }
  __syncthreads();
  if (tid < kMaxBlocks) {
    for (int w = 0; w < warp; ++w) rows += s_warp[w];
    s_end[tid] = rows;
  }
  __syncthreads();
  const int all = s_end[kMaxBlocks - 1];
  for (int u = warp * gridDim.x + blockIdx.x; u < all; u += gridDim.x * (kJoinThreads / 32)) {
    int lo = 0, hi = kMaxBlocks - 1;  // the first tile that ends after row u
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (s_end[mid] > u) hi = mid;
      else lo = mid + 1;
    }
    const CutTile cut = s_cut[lo];
    const int r = u - (lo ? s_end[lo - 1] : 0), tk = r / p.G, g = r - tk * p.G;
    const int row = (tk >= p.TT ? 128 + (tk - p.TT) * p.G : tk * p.G) + g;
    const long tok = cut.tok0 + tk;
    const int head = cut.hv * p.G + g;
    join_row<DH, 4>(part_count(cut.parts), [&](int i) { return p.slot_ml + part_row(cut.parts, i, row, blocks) * 2; },
                 [&](int i) { return p.slots + part_row(cut.parts, i, row, blocks) * DH; }, p.o + tok * p.ldo + (long)head * DH,
                 p.lse != nullptr ? p.lse + tok * p.H + head : nullptr);
  }
}

// Every row of a batch that shares a prefix: its own parts and the prefix's. A whole tile's part lies
// in the row buffers, a cut one's in the slots, at the row's place inside its tile.
template <int DH>
__global__ void __launch_bounds__(kJoinThreads) join_rows_kernel(PackedAttnParams p, int blocks) {
  wait_for_earlier_kernels();
  let_later_kernels_start();
  const long cls = (long)p.N * p.H, orow = (long)blockIdx.x * (kJoinThreads / 32) + (threadIdx.x >> 5);
  if (orow >= cls) return;
  const int failed = *p.err, own = p.row_parts[orow], pre = p.row_parts[cls + orow];
  const int from = p.q_start[0], to = p.q_start[p.B];
  const int tok = static_cast<int>(orow / p.H), head = static_cast<int>(orow - (long)tok * p.H);
  if ((failed != 0) | (tok < from) | (tok >= to)) return;  // no parts; no request's row (five reads at once)
  auto whole = [](int parts) { return (parts & 0xffffff) == kWholeRow; };
  const int n_own = whole(own) ? 1 : part_count(own), n_pre = whole(pre) ? 1 : part_count(pre);
  const int own_row = static_cast<unsigned>(own) >> 24, pre_row = static_cast<unsigned>(pre) >> 24;
  join_row<DH, 8>(n_own + n_pre,
               [&](int i) -> const float* {
                 if (i < n_own) return whole(own) ? p.row_ml + orow * 2 : p.slot_ml + part_row(own, i, own_row, blocks) * 2;
                 return whole(pre) ? p.row_ml + (cls + orow) * 2 : p.slot_ml + part_row(pre, i - n_own, pre_row, blocks) * 2;
               },
               [&](int i) -> const float* {
                 if (i < n_own) return whole(own) ? p.row_o + orow * DH : p.slots + part_row(own, i, own_row, blocks) * DH;
                 return whole(pre) ? p.row_o + (cls + orow) * DH : p.slots + part_row(pre, i - n_own, pre_row, blocks) * DH;
               },
               p.o + (long)tok * p.ldo + (long)head * DH, p.lse != nullptr ? p.lse + orow : nullptr);
}

template <int DH>
void launch(const CUtensorMap& q, const CUtensorMap& q1, const CUtensorMap& k, const CUtensorMap& v,
            const PackedAttnParams& p, cudaStream_t stream) {
  constexpr int smem = Cfg<DH>::SMEM + Cfg<DH>::TAIL;
  static_assert(smem <= 232448, "shared memory of a block");
  static std::atomic<uint64_t> prepared{0};  // devices whose kernel may use that much
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 64 || !(prepared.load(std::memory_order_relaxed) >> dev & 1)) {
    cudaFuncSetAttribute(packed_attention_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (dev < 64) prepared.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
  }
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const int blocks = packed_attention_blocks();
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchKernelEx(&cfg, packed_attention_kernel<DH>, q, q1, k, v, p);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  if (p.row_o != nullptr) {
    const long per = kJoinThreads / 32;
    cfg.gridDim = dim3(static_cast<unsigned>(((long)p.N * p.H + per - 1) / per));
    cudaLaunchKernelEx(&cfg, join_rows_kernel<DH>, p, blocks);
  } else {
    cfg.gridDim = dim3(kCutBlocksPerSm * blocks);
    cudaLaunchKernelEx(&cfg, join_cut_tiles_kernel<DH>, p, blocks);
  }
}

}  // namespace

int packed_attention_blocks() {
  static int sms[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev] < kMaxBlocks ? sms[dev] : kMaxBlocks;
}

void launch_packed_attention(int head_dim, const CUtensorMap& q, const CUtensorMap& q1, const CUtensorMap& k,
                             const CUtensorMap& v, const PackedAttnParams& p, cudaStream_t stream) {
  if (head_dim == 128) launch<128>(q, q1, k, v, p, stream);
  else launch<64>(q, q1, k, v, p, stream);
}

}  // namespace appcorr
