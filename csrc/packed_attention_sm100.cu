// Packed causal grouped-query attention on the 5th-generation tensor cores (tcgen05 + TMEM + TMA).
//
//   o_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = 2^(c q_t . k_j - c max_j),   c = scale log2 e,
// for the tokens t of every request and the keys j <= kv_len - q_len + t of its cache.
//
// Tile. The G query heads that share a key head are rows of one tile (row = token * G + head), so a
// key block is read once for all of them and one decoding token fills G rows instead of one. A tile
// is two halves of 128 rows (floor(128 / G) tokens each) against key blocks of 128, the page size;
// S = Q K^T and P V run with fp32 accumulators in TMEM: S0 S1 | O0 O1, 128 columns each. The two
// halves are worked in turn, so that the tensor core has one half's products to do while the
// other half is in its softmax:
//   warp 0      walks the work list, publishes tiles, TMA of Q and of a ring of K / V tiles
//   warp 1      MMA: PV0_j S0_{j+1} PV1_j S1_{j+1}; P is read from TMEM, where it replaces its S
//   warps 4..7  softmax of half 0, warps 8..11 of half 1, one row per thread: running maximum and
//               sum in fp32, P rounded to bf16 (the tensor core's operand type; its error is a
//               relative 2^-8 of each probability, averaged over the keys), O rescaled in TMEM only
//               when the maximum has grown by 2^8 since it was last applied (P <= 2^8, exact at the
//               end because the sum carries the same factor)
// MMAs of one thread complete in order: S_j's commit also means that PV_{j-1} has completed, so a
// softmax warp that has S_j may rescale O, and S_{j+1} may overwrite P_j once PV_j was issued.
//
// Work list. All tiles' costs (visible keys plus kTileCost for a tile's own start and end) are laid
// on one line, ordered by request, key head and tile; every block takes an equal stretch of it, so a
// stretch may begin and end inside a tile, on a key block. That balances prompts of any mix of
// lengths and splits few long rows over all SMs by the same rule, without a host that knows the
// lengths: a block sums the costs of all requests itself, and positions inside a request have a
// closed form. A tile cut by a stretch's end leaves partial results (O, max, sum in fp32); the
// warp that arrives last at its 32 rows joins them in order, so the result does not depend on
// which one that is. Nothing waits for another block.
//
// Keys past a request's end in its last page may hold anything: their scores are replaced, and
// their V rows are zeroed in shared memory, since 0 * NaN would reach the accumulators.
// All waits are bounded; a wait that runs out sets the error word and every role leaves.
#include "packed_attention.h"

#include "sm100_common.cuh"

namespace appcorr {
namespace {

using bf16 = __nv_bfloat16;

constexpr int kThreads = 384;      // three warpgroups: roles, softmax of half 0, softmax of half 1
constexpr int kTiles = 4;          // published tiles in flight
constexpr int kBlk = 128;         // keys per block = rows per page
constexpr long kTileCost = 128;   // a tile's fixed cost, in keys
constexpr long kLeastWork = 256;  // least work of a block, in the same unit

template <int DH>
struct Cfg {
  static constexpr int NCH = DH / 64;                       // 64-column chunks
  static constexpr uint32_t CHUNK = 128 * 128;              // one [128 rows x 64] bf16 box
  static constexpr uint32_t TILE = NCH * CHUNK;             // K or V block, or half of Q
  static constexpr int NST = DH == 128 ? 5 : 8;             // ring of K / V blocks
  static constexpr uint32_t SMEM = 2 * TILE + NST * TILE;
  static constexpr uint32_t TAIL = 2048;  // barriers, tiles, scan (under 1 KB), and what aligns the base to 1 KB
};

struct Tile {
  int tok0, ntok;  // first packed row and number of tokens
  int lim0;        // last key visible to its first token
  int kv;          // keys of the request
  int hv;          // key head * sub-groups + sub-group
  int jb, n0, n1;  // first key block of this stretch, key blocks of each half
  int flags;       // 1: whole tile (direct output), 2: end of the work
  int slot, first, expect;
  int nb;
  long at, cost;   // place and length on the work line
};

struct Request {
  int q0, q, past, kv, nt;
  long base;  // cost of a tile before its own new tokens
  int slope;  // more keys per tile (0: every token sees all keys)
};

template <bool PREFIX>
__device__ __forceinline__ Request make_request(const PackedAttnParams& p, int q0, int q1, int kv) {
  Request r;
  q0 = max(q0, 0);
  q1 = min(q1, p.N);
  r.q0 = q0;
  r.q = max(q1 - q0, 0);
  r.kv = max(kv, 0);
  r.past = r.kv - r.q;
  const int tt2 = 2 * p.TT;
  r.nt = (r.q + tt2 - 1) / tt2;
  r.base = kTileCost + (PREFIX ? r.kv : max(r.past, 0));
  r.slope = PREFIX ? 0 : tt2;
  return r;
}
template <bool PREFIX>
__device__ __forceinline__ Request load_request(const PackedAttnParams& p, int b) {
  if (PREFIX) return make_request<PREFIX>(p, 0, p.q_start[p.B], p.shared_len);
  return make_request<PREFIX>(p, p.q_start[b], p.q_start[b + 1], p.kv_len[b]);
}
// cost of the first k tiles of one head
__device__ __forceinline__ long tiles_cost(const Request& r, int k) {
  long c = k * r.base + (long)r.slope * k * (k + 1) / 2;
  if (k == r.nt && r.slope) c -= (long)r.nt * r.slope - r.q;
  return c;
}
// key blocks before point w of the line inside the tile [at, at + cost)
__device__ __forceinline__ int cut_block(long w, long at, long cost, int nb) {
  if (w <= at) return 0;
  if (w >= at + cost) return nb;
  const long s = (w - at - kTileCost + kBlk / 2) / kBlk;
  return static_cast<int>(min(max(s, 0L), static_cast<long>(nb)));
}
__device__ __forceinline__ long stretch(long W, int c, int n) { return W * c / n; }

__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, int* err, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, code));
}

template <int DH, bool PREFIX>
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
  uint64_t* s_full = bars + 2;    // 2
  uint64_t* p_full = bars + 4;    // 2
  uint64_t* o_full = bars + 6;    // 2
  uint64_t* o_empty = bars + 8;   // 2
  uint64_t* t_full = bars + 10;           // kTiles
  uint64_t* t_empty = t_full + kTiles;    // kTiles
  uint64_t* done = t_empty + kTiles;
  uint64_t* full = done + 1;              // NST
  uint64_t* empty = full + NST;           // NST
  Tile* tiles = reinterpret_cast<Tile*>(bars + 40);
  long* scan = reinterpret_cast<long*>(tiles + kTiles);  // the warps' sums, the begin's offset
  int* s_int = reinterpret_cast<int*>(scan + kThreads / 32 + 1);  // begin's request, TMEM base

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // ---------------------------------------------------------------- this block's stretch of the line
  const int B = PREFIX ? 1 : p.B;
  long sum = 0;
  for (int b = tid; b < B; b += kThreads) {
    const Request r = load_request<PREFIX>(p, b);
    sum += p.Hv * tiles_cost(r, r.nt);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) scan[warp] = sum;
  __syncthreads();
  long W = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) W += scan[w];
  if (W == 0) return;
  const int n = static_cast<int>(min(max(W / kLeastWork, 1L), static_cast<long>(gridDim.x)));
  const int me = blockIdx.x;
  if (me >= n) return;
  const long w0 = stretch(W, me, n), w1 = stretch(W, me + 1, n);
  long base = 0;
  for (int b0 = 0; b0 < B; b0 += kThreads) {
    __syncthreads();
    const int b = b0 + tid;
    long v = 0;
    if (b < B) {
      const Request r = load_request<PREFIX>(p, b);
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
    if (before + inc - v <= w0 && w0 < before + inc) {
      s_int[0] = b;
      scan[kThreads / 32] = w0 - (before + inc - v);
    }
    base += all;
    if (base > w0) break;
  }

  if (warp == 0 && lane == 0) {
    mbar_init(smem_addr(q_full), 1);
    mbar_init(smem_addr(q_empty), 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&s_full[i]), 1);
      mbar_init(smem_addr(&p_full[i]), 4);
      mbar_init(smem_addr(&o_full[i]), 1);
      mbar_init(smem_addr(&o_empty[i]), 4);
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_int[1];

  // registers: 384 threads start with 168 each (64512); the roles keep 88, the softmax threads get
  // 208 (128 x (88 + 208 + 208) = 64512)
  if (warp < 4) {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  if (warp == 0) {
    // ------------------------------------------------------------------------------ work list + TMA
    bool ok = true;
    int b = s_int[0];
    Request r = load_request<PREFIX>(p, b);
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
    int nq = 0, np = 0;
    while (ok && at < w1) {
      const long cost = tiles_cost(r, t + 1) - tiles_cost(r, t);
      const int t0 = t * tt2, ntok = min(tt2, r.q - t0);
      const int vis1 = PREFIX ? r.kv : min(max(r.past + t0 + ntok, 0), r.kv);
      const int vis0 = PREFIX ? r.kv : min(max(r.past + t0 + min(ntok, p.TT), 0), r.kv);
      const int nb = (vis1 + kBlk - 1) / kBlk, nb0 = (vis0 + kBlk - 1) / kBlk;
      const bool owner = at >= w0;
      const int jb = cut_block(w0, at, cost, nb), je = cut_block(w1, at, cost, nb);
      if (je > jb || (nb == 0 && owner)) {
        Tile tl;
        tl.tok0 = r.q0 + t0;
        tl.ntok = ntok;
        tl.lim0 = PREFIX ? r.kv : r.past + t0;
        tl.kv = r.kv;
        tl.hv = hv;
        tl.jb = jb;
        tl.n0 = min(max(nb0 - jb, 0), je - jb);
        tl.n1 = ntok > p.TT ? je - jb : 0;
        const bool whole = jb == 0 && je == nb;
        tl.flags = whole ? 1 : 0;
        tl.nb = nb;
        tl.at = at;
        tl.cost = cost;
        tl.slot = owner ? 2 * me + 1 : 2 * me;
        tl.first = me;
        tl.expect = 0;
        if (!whole) {  // the blocks that share this tile: those whose stretch meets [at, at + cost)
          const int c0 = static_cast<int>(((at + 1) * n + W - 1) / W) - 1;
          const int c1 = static_cast<int>(((at + cost) * n + W - 1) / W) - 1;
          int cnt = 0;
          for (int c = c0 + lane; c <= c1; c += 32)
            cnt += cut_block(stretch(W, c + 1, n), at, cost, nb) > cut_block(stretch(W, c, n), at, cost, nb);
          tl.expect = __reduce_add_sync(0xffffffffu, cnt);
          tl.first = c0;
        }
        ok = warp_wait(smem_addr(&t_empty[np % kTiles]), ((np / kTiles) & 1) ^ 1, p.err, kErrTimeoutProducer);
        if (!ok) break;
        if (lane == 0) {
          tiles[np % kTiles] = tl;
          mbar_arrive(smem_addr(&t_full[np % kTiles]));
        }
        ++np;
        const int kvh = hv / p.ng;
        int pg = 0;
        for (int j = 0; ok && j < je - jb; ++j) {
          const int blk = jb + j;
          int row;
          if (PREFIX || p.table != nullptr) {
            if ((j & 31) == 0) {
              const int e = blk + lane;
              pg = e < p.W && j + lane < je - jb ? p.table[(PREFIX ? 0 : b * p.ld_table) + e] : -1;
              if (pg < 0 || pg >= p.pages) pg = p.pages;  // no page: past the pool, where TMA fills zeros
            }
            row = __shfl_sync(0xffffffffu, pg, j & 31) * kBlk;
          } else {
            const int k0 = p.k_start[b];
            row = k0 >= 0 && k0 < p.key_rows ? k0 + blk * kBlk : p.key_rows;
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
          do {
            if (++b >= B) break;
            r = load_request<PREFIX>(p, b);
          } while (r.nt == 0);
          if (b >= B) break;
        }
      }
    }
    ok = ok && warp_wait(smem_addr(&t_empty[np % kTiles]), ((np / kTiles) & 1) ^ 1, p.err, kErrTimeoutProducer);
    if (ok && lane == 0) {
      tiles[np % kTiles].flags = 2;
      mbar_arrive(smem_addr(&t_full[np % kTiles]));
    }
    if (!ok) {  // let the copies in flight land before the block ends
      const uint32_t from = it > NST ? it - NST : 0;
      for (uint32_t i = from; i < it; ++i) mbar_wait(smem_addr(&full[i % NST]), (i / NST) & 1, nullptr, 0);
      if (nq) mbar_wait(smem_addr(q_full), (nq - 1) & 1, nullptr, 0);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------------------------ MMA
    bool ok = true;
    uint32_t it = 0;
    int nq = 0;
    int np_[2] = {0, 0}, no_[2] = {0, 0};  // P tiles and O tiles consumed per half
    const uint32_t qa = smem_addr(sQ), kva = smem_addr(sKV);
    auto issue_s = [&](int hf, uint32_t i) {
      if (lane == 0) {
        const uint32_t ka = kva + (i % NST) * C::TILE, qh = qa + hf * C::TILE;
#pragma unroll
        for (int k = 0; k < DH / 16; ++k) {
          const uint32_t off = (k >> 2) * C::CHUNK + (k & 3) * 32;
          umma_f16(tmem + hf * 128, sw128_kmajor_desc(qh + off), sw128_kmajor_desc(ka + off), IDESC_S, k > 0);
        }
        umma_commit(smem_addr(&s_full[hf]));
      }
    };
    for (int np = 0;; ++np) {
      ok = warp_wait(smem_addr(&t_full[np % kTiles]), (np / kTiles) & 1, p.err, kErrTimeoutMma);
      if (!ok) break;
      const Tile& tl = tiles[np % kTiles];
      const int flags = tl.flags, nn[2] = {tl.n0, tl.n1}, kv = tl.kv, jb = tl.jb;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&t_empty[np % kTiles]));
      if (flags & 2) break;
      const int cnt = max(nn[0], nn[1]);
      if (cnt == 0) continue;
      ok = warp_wait(smem_addr(&full[it % NST]), (it / NST) & 1, p.err, kErrTimeoutMma) &&
           warp_wait(smem_addr(q_full), nq & 1, p.err, kErrTimeoutMma);
      if (!ok) break;
      ++nq;
      tc_fence_after();
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        if (nn[hf] > 0) issue_s(hf, it);
      if (lane == 0) {
        umma_commit(smem_addr(&empty[it % NST]));
        if (cnt == 1) umma_commit(smem_addr(q_empty));
      }
      ++it;
      for (int j = 0; ok && j < cnt; ++j) {
        const uint32_t iv = it, ik = it + 1;
        const bool more = j + 1 < cnt;
        ok = warp_wait(smem_addr(&full[iv % NST]), (iv / NST) & 1, p.err, kErrTimeoutMma);
        if (!ok) break;
        const int live = kv - (jb + j) * kBlk;  // keys of this block that exist
        if (live < kBlk) {
          for (int i = lane; i < (kBlk - live) * 8; i += 32)
#pragma unroll
            for (int c = 0; c < NCH; ++c)
              *reinterpret_cast<uint4*>(sKV + (iv % NST) * C::TILE + c * C::CHUNK + live * 128 + i * 16) = make_uint4(0, 0, 0, 0);
          fence_proxy_async_smem();
          __syncwarp();
        }
        if (more) ok = warp_wait(smem_addr(&full[ik % NST]), (ik / NST) & 1, p.err, kErrTimeoutMma);
        if (!ok) break;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          if (j >= nn[hf]) continue;
          ok = warp_wait(smem_addr(&p_full[hf]), np_[hf] & 1, p.err, kErrTimeoutMma);
          if (!ok) break;
          ++np_[hf];
          if (j == 0) {
            ok = warp_wait(smem_addr(&o_empty[hf]), (no_[hf] & 1) ^ 1, p.err, kErrTimeoutMma);
            if (!ok) break;
            ++no_[hf];
          }
          tc_fence_after();
          if (lane == 0) {
            const uint32_t va = kva + (iv % NST) * C::TILE;
#pragma unroll
            for (int k = 0; k < kBlk / 16; ++k)
              umma_f16_tmem_a(tmem + O_COL + hf * 128, tmem + hf * 128 + k * 8, sw128_mnmajor_desc(va + k * 2048, C::CHUNK, 1024),
                              IDESC_O, (j > 0 || k > 0) ? 1u : 0u);
            if (j + 1 == nn[hf]) umma_commit(smem_addr(&o_full[hf]));
          }
          if (j + 1 < nn[hf]) issue_s(hf, ik);
        }
        if (!ok) break;
        if (lane == 0) {
          umma_commit(smem_addr(&empty[iv % NST]));
          if (more) {
            umma_commit(smem_addr(&empty[ik % NST]));
            if (j + 2 == cnt) umma_commit(smem_addr(q_empty));
          }
        }
        it += more ? 2 : 1;
      }
      if (!ok) break;
    }
    if (!ok) {  // products in flight end before TMEM is given back
      if (lane == 0) umma_commit(smem_addr(done));
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
    int ns = 0, no = 0;
    bool ok = true;
    for (int np = 0;; ++np) {
      ok = warp_wait(smem_addr(&t_full[np % kTiles]), (np / kTiles) & 1, p.err, kErrTimeoutEpilogue);
      if (!ok) break;
      const Tile& tl = tiles[np % kTiles];
      if (tl.flags & 2) break;
      auto release = [&] {  // this warp no longer reads the tile's description
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&t_empty[np % kTiles]));
      };
      const int cnt = hf ? tl.n1 : tl.n0;
      const int tk = hf * p.TT + rtok;
      const bool valid = rtok < p.TT && tk < tl.ntok;
      const bool alive = __any_sync(0xffffffffu, valid);  // some row of this warp is stored
      const int klim = PREFIX ? tl.kv - 1 : min(tl.kv - 1, tl.lim0 + tk);
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
          const int over = klim - (tl.jb + j) * kBlk;  // last visible key of this block
          if (__any_sync(0xffffffffu, over < kBlk - 1)) {
#pragma unroll
            for (int i = 0; i < kBlk; ++i) sv[i] = i <= over ? sv[i] : -INFINITY;
          }
          float mx[4] = {sv[0], sv[1], sv[2], sv[3]};
#pragma unroll
          for (int i = 4; i < kBlk; ++i) mx[i & 3] = fmaxf(mx[i & 3], sv[i]);
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
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
          float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float e0 = ex2_approx(fmaf(sv[c * 64 + 2 * i], sl2, -moff));
              const float e1 = ex2_approx(fmaf(sv[c * 64 + 2 * i + 1], sl2, -moff));
              ls[(2 * i) & 3] += e0;
              ls[(2 * i + 1) & 3] += e1;
              pk[i] = pack_bf16x2(e0, e1);
            }
            tmem_st32(s_addr + c * 32, pk);
          }
          l_run += (ls[0] + ls[1]) + (ls[2] + ls[3]);
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_addr(&p_full[hf]));
      }
      if (!ok) break;
      if (cnt > 0) {
        ok = warp_wait(smem_addr(&o_full[hf]), no & 1, p.err, kErrTimeoutEpilogue);
        if (!ok) break;
        ++no;
        tc_fence_after();
      }
      const bool has = hf == 0 || tl.ntok > p.TT;
      if (!has || !alive) {
        if (cnt > 0) {
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&o_empty[hf]));
        }
        release();
        continue;
      }
      const long tok = tl.tok0 + tk;
      const int head = tl.hv * p.G + rhead;
      const float mlog = m_run == -INFINITY ? -INFINITY : m_run * sl2;  // max in log2 units
      if (tl.flags & 1) {
        float w_own = l_run > 0.f || l_run != l_run ? 1.f / l_run : 0.f, w_pri = 0.f;
        float lse2 = mlog + log2f(l_run);
        const long orow = tok * p.H + head;
        if (!PREFIX && p.prior != nullptr && valid) {  // join the prefix's result
          const float lp = p.prior_lse[orow];
          const float top = fmaxf(mlog, lp), safe = top == -INFINITY ? 0.f : top;
          const float a = exp2f(mlog - safe), c = exp2f(lp - safe), total = a * l_run + c;
          w_own = total > 0.f || total != total ? a / total : 0.f;
          w_pri = total > 0.f || total != total ? c / total : 0.f;
          lse2 = safe + log2f(total);
        }
#pragma unroll 1
        for (int c = 0; c < DH / 32; ++c) {
          uint32_t u[32];
          __syncwarp();
          if (cnt > 0) {
            tmem_ld32(o_addr + c * 32, u);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = 0u;
          }
          if (valid) {
            float x[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(u[i]) * w_own;
            if (PREFIX) {
              float4* dst = reinterpret_cast<float4*>(p.prior + orow * DH + c * 32);
#pragma unroll
              for (int i = 0; i < 8; ++i) dst[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            } else {
              if (p.prior != nullptr) {
                const float4* src = reinterpret_cast<const float4*>(p.prior + orow * DH + c * 32);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float4 f = src[i];
                  x[4 * i] = fmaf(f.x, w_pri, x[4 * i]);
                  x[4 * i + 1] = fmaf(f.y, w_pri, x[4 * i + 1]);
                  x[4 * i + 2] = fmaf(f.z, w_pri, x[4 * i + 2]);
                  x[4 * i + 3] = fmaf(f.w, w_pri, x[4 * i + 3]);
                }
              }
              uint4* dst = reinterpret_cast<uint4*>(p.o + tok * p.ldo + (long)head * DH + c * 32);
#pragma unroll
              for (int i = 0; i < 4; ++i)
                dst[i] = make_uint4(pack_bf16x2(x[8 * i], x[8 * i + 1]), pack_bf16x2(x[8 * i + 2], x[8 * i + 3]),
                                    pack_bf16x2(x[8 * i + 4], x[8 * i + 5]), pack_bf16x2(x[8 * i + 6], x[8 * i + 7]));
            }
          }
        }
        if (valid) {
          if (PREFIX) p.prior_lse[orow] = lse2;
          else if (p.lse != nullptr) p.lse[orow] = lse2 * 0.69314718055994531f;
        }
        if (cnt > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&o_empty[hf]));
        }
        release();
        continue;
      }
      // -------- a cut tile: leave this stretch's part, join them all if this warp is the last to come
      {
        const long srow = (long)tl.slot * kPaRows + hf * 128 + row;
#pragma unroll 1
        for (int c = 0; c < DH / 32; ++c) {
          uint32_t u[32];
          __syncwarp();
          if (cnt > 0) {
            tmem_ld32(o_addr + c * 32, u);
            tmem_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) u[i] = 0u;
          }
          if (valid) {
            uint4* dst = reinterpret_cast<uint4*>(p.slots + srow * DH + c * 32);
#pragma unroll
            for (int i = 0; i < 8; ++i) dst[i] = make_uint4(u[4 * i], u[4 * i + 1], u[4 * i + 2], u[4 * i + 3]);
          }
        }
        if (valid) *reinterpret_cast<float2*>(p.slot_ml + srow * 2) = make_float2(mlog, l_run);
        if (cnt > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&o_empty[hf]));
        }
        __threadfence();
        __syncwarp();
        int* counter = p.counters + tl.first * 8 + hf * 4 + qd;
        int old = 0;
        if (lane == 0) old = atomicAdd(counter, 1);
        old = __shfl_sync(0xffffffffu, old, 0);
        if (old != tl.expect - 1) {
          release();
          continue;
        }
        if (lane == 0) *counter = 0;
        __threadfence();
        const unsigned rows = __ballot_sync(0xffffffffu, valid);
        constexpr int CPL = DH / 32;  // columns per lane
        const int c_last = static_cast<int>(((tl.at + tl.cost) * n + W - 1) / W) - 1;
        for (int rr = 0; rr < 32; ++rr) {
          if (!((rows >> rr) & 1)) continue;
          const int r_abs = hf * 128 + qd * 32 + rr;
          const long rtk = __shfl_sync(0xffffffffu, (int)tok, rr);
          const int rhd = __shfl_sync(0xffffffffu, head, rr);
          const long orow = rtk * p.H + rhd;
          float acc[CPL], top = -INFINITY, total = 0.f;
#pragma unroll
          for (int i = 0; i < CPL; ++i) acc[i] = 0.f;
          if (!PREFIX && p.prior != nullptr) {
            top = p.prior_lse[orow];
            total = top == -INFINITY ? 0.f : 1.f;
#pragma unroll
            for (int i = 0; i < CPL; ++i) acc[i] = p.prior[orow * DH + lane * CPL + i] * total;
          }
          for (int cb = tl.first; cb <= c_last; cb += 32) {
            const int c = cb + lane;
            const bool part = c <= c_last && cut_block(stretch(W, c + 1, n), tl.at, tl.cost, tl.nb) >
                                                 cut_block(stretch(W, c, n), tl.at, tl.cost, tl.nb);
            const long srow2 = (long)(c == tl.first ? 2 * c + 1 : 2 * c) * kPaRows + r_abs;
            float2 ml = make_float2(-INFINITY, 0.f);
            if (part) ml = __ldcg(reinterpret_cast<const float2*>(p.slot_ml + srow2 * 2));
            float mt = ml.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
            mt = fmaxf(mt, top);
            const float safe = mt == -INFINITY ? 0.f : mt;
            const float old_w = exp2f(top - safe), w = part ? exp2f(ml.x - safe) : 0.f;
            top = mt;
            float part_sum = w * ml.y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) part_sum += __shfl_xor_sync(0xffffffffu, part_sum, o);
            total = total * old_w + part_sum;
#pragma unroll
            for (int i = 0; i < CPL; ++i) acc[i] *= old_w;
            unsigned parts = __ballot_sync(0xffffffffu, part);
            while (parts) {
              const int src = __ffs(parts) - 1;
              parts &= parts - 1;
              const float ws = __shfl_sync(0xffffffffu, w, src);
              const long sr = (long)(cb + src == tl.first ? 2 * (cb + src) + 1 : 2 * (cb + src)) * kPaRows + r_abs;
              const float* f = p.slots + sr * DH + lane * CPL;
#pragma unroll
              for (int i = 0; i < CPL; ++i) acc[i] = fmaf(ws, __ldcg(f + i), acc[i]);
            }
          }
          const float inv = total > 0.f || total != total ? 1.f / total : 0.f;
          const float lse2 = top == -INFINITY ? -INFINITY : top + log2f(total);
          if (PREFIX) {
#pragma unroll
            for (int i = 0; i < CPL; ++i) p.prior[orow * DH + lane * CPL + i] = acc[i] * inv;
            if (lane == 0) p.prior_lse[orow] = lse2;
          } else {
#pragma unroll
            for (int i = 0; i < CPL; i += 2)
              *reinterpret_cast<uint32_t*>(p.o + rtk * p.ldo + (long)rhd * DH + lane * CPL + i) =
                  pack_bf16x2(acc[i] * inv, acc[i + 1] * inv);
            if (lane == 0 && p.lse != nullptr) p.lse[orow] = lse2 * 0.69314718055994531f;
          }
        }
        release();
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

template <int DH, bool PREFIX>
void launch(const CUtensorMap& q, const CUtensorMap& q1, const CUtensorMap& k, const CUtensorMap& v,
            const PackedAttnParams& p, cudaStream_t stream) {
  constexpr int smem = Cfg<DH>::SMEM + Cfg<DH>::TAIL;
  auto kern = packed_attention_kernel<DH, PREFIX>;
  cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  kern<<<packed_attention_blocks(), kThreads, smem, stream>>>(q, q1, k, v, p);
}

}  // namespace

int packed_attention_blocks() {
  static int sms[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return 148;
  if (sms[dev] == 0) cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev);
  return sms[dev];
}

void launch_packed_attention(int head_dim, bool prefix_pass, const CUtensorMap& q, const CUtensorMap& q1,
                             const CUtensorMap& k, const CUtensorMap& v, const PackedAttnParams& p, cudaStream_t stream) {
  if (head_dim == 128) {
    if (prefix_pass) launch<128, true>(q, q1, k, v, p, stream);
    else launch<128, false>(q, q1, k, v, p, stream);
  } else {
    if (prefix_pass) launch<64, true>(q, q1, k, v, p, stream);
    else launch<64, false>(q, q1, k, v, p, stream);
  }
}

}  // namespace appcorr
