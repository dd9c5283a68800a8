// Block tables and slot maps of a packed batch, built on the device from request lengths.
//
// Request b brings q_len[b] new tokens after past[b] cached ones. With pages of 128 rows,
//   q_start    = exclusive prefix sums of q_len                      kv_len[b] = past[b] + q_len[b]
//   have[b]    = ceil(past[b] / 128)      need[b] = min(ceil(kv_len[b] / 128), W) - have[b]
//   first[b]   = exclusive prefix sums of need
//   table[b, have[b] + i] = free_pages[free_start + first[b] + i]    (i < need[b]; -1 past the list)
//   token n = q_start[b] + i:  req = b, pos = past[b] + i, row = page(pos / 128) * 128 + pos % 128
// and free_next = (first free index after this step, pages that could not be given).
//
// Nothing but latency bounds it (12 bytes a token out: the 224k tokens of 2048 requests are 2.7 MB and take
// 6.4 us, one request's token 2.9 us), so it is ONE launch in which no block waits for another: every
// block scans all the requests itself, 1024 at a time in shared memory; block k then owns an equal
// share of the tokens (request found by a binary search in shared memory) and every gridDim-th
// request's new pages. A token in a page of this step takes the page from the free list, not from the
// table. (Two launches, or a look-back between the blocks, were not built.)
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "checks.h"
#include "registry.h"

namespace appcorr {

constexpr int kPlRows = 128;      // rows per cache page
constexpr int kPlThreads = 1024;  // requests scanned at a time
constexpr unsigned kPlPages = (1u << 31) / kPlRows;  // pages whose rows have 32-bit numbers

struct LayoutParams {
  const int* q_len;
  const int* past;
  int* table;
  long ld_table;
  const int* free_pages;
  const int* free_start;
  int* q_start;
  int* kv_len;
  int* rows;
  int* req;
  int* pos;
  int* free_next;
  int B, W, F, N;
};

// past + q_len passes 31 bits where a length is near 2^31, and is kept in unsigned 32 bits
__device__ __forceinline__ int blocks_of(unsigned rows) { return static_cast<int>(rows / kPlRows + (rows % kPlRows != 0)); }
__device__ __forceinline__ int capped(unsigned n) { return static_cast<int>(min(n, 0x7fffffffu)); }

__global__ void __launch_bounds__(kPlThreads) packed_layout_kernel(LayoutParams p) {
  __shared__ int s_start[kPlThreads + 1], s_past[kPlThreads], s_first[kPlThreads];
  __shared__ int s_warp[3][32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int share = (p.N + gridDim.x - 1) / gridDim.x;
  const int n0 = min(p.N, share * (int)blockIdx.x), n1 = min(p.N, n0 + share);
  const int begin = max(*p.free_start, 0);
  int tok_base = 0, page_base = 0, over_base = 0;  // sums over the chunks before this one
  for (int b0 = 0; b0 < p.B; b0 += kPlThreads) {
    const int b = b0 + tid, nb = min(kPlThreads, p.B - b0);
    const int q = b < p.B ? max(p.q_len[b], 0) : 0, past = b < p.B ? max(p.past[b], 0) : 0;
    const int have = blocks_of(past), total = blocks_of((unsigned)past + q);
    const int need = max(min(total, p.W) - have, 0), over = max(total - max(p.W, have), 0);
    // three inclusive scans at once: tokens, new pages, blocks past the table's width
    int v[3] = {q, need, over};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int up = __shfl_up_sync(0xffffffffu, v[k], o);
        if (lane >= o) v[k] += up;
      }
    }
    if (lane == 31) {
#pragma unroll
      for (int k = 0; k < 3; ++k) s_warp[k][warp] = v[k];
    }
    __syncthreads();
    if (warp < 3) {
      int w = s_warp[warp][lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += up;
      }
      s_warp[warp][lane] = w;
    }
    __syncthreads();
    const int before = warp ? s_warp[0][warp - 1] : 0;
    const int tok = tok_base + before + v[0] - q;                                  // this request's first token
    const int first = page_base + (warp ? s_warp[1][warp - 1] : 0) + v[1] - need;  // its first new page
    s_start[tid] = tok;
    s_past[tid] = past;
    s_first[tid] = first;
    const int tok_end = tok_base + s_warp[0][31];
    const int page_end = page_base + s_warp[1][31], over_end = over_base + s_warp[2][31];
    if (tid == 0) s_start[nb] = tok_end;
    if (blockIdx.x == 0 && b < p.B) {
      p.q_start[b] = tok;
      p.kv_len[b] = capped((unsigned)past + q);
    }
    __syncthreads();
    // new pages of this block's requests: one warp each
    for (int r = blockIdx.x + gridDim.x * warp; r < nb; r += gridDim.x * (kPlThreads / 32)) {
      const unsigned pst = s_past[r], ql = (unsigned)s_start[r + 1] - s_start[r];
      const int hv = blocks_of(pst);
      const int nd = min(blocks_of(pst + ql), p.W) - hv;
      for (int i = lane; i < nd; i += 32) {
        const unsigned long src = (long)begin + s_first[r] + i;
        p.table[(b0 + r) * p.ld_table + hv + i] = src < p.F ? p.free_pages[src] : -1;
      }
    }
    // this block's tokens inside the chunk
    for (int n = max(n0, min(tok_base, n1)) + tid; n < min(n1, tok_end); n += kPlThreads) {
      int lo = 0, hi = nb;  // the last request that starts at or before n (empty ones lie before it)
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= n) lo = mid;
        else hi = mid;
      }
      const unsigned pst = s_past[lo], at = pst + n - s_start[lo];
      const int blk = at / kPlRows, hv = blocks_of(pst);
      int page = -1;
      if (blk < p.W) {
        if (blk < hv) {
          page = p.table[(b0 + lo) * p.ld_table + blk];
        } else {
          const unsigned long src = (long)begin + s_first[lo] + blk - hv;
          if (src < p.F) page = p.free_pages[src];
        }
      }
      p.rows[n] = static_cast<unsigned>(page) < kPlPages ? page * kPlRows + at % kPlRows : -1;
      p.req[n] = b0 + lo;
      p.pos[n] = capped(at);
    }
    tok_base = tok_end;
    page_base = page_end;
    over_base = over_end;
    __syncthreads();
  }
  for (int n = max(n0, min(tok_base, n1)) + tid; n < n1; n += kPlThreads) p.rows[n] = p.req[n] = p.pos[n] = -1;  // padding
  if (blockIdx.x == 0 && tid == 0) {
    p.q_start[p.B] = tok_base;
    const long end = (long)begin + page_base, given = min(end, (long)max(p.F, begin));
    p.free_next[0] = static_cast<int>(given);
    p.free_next[1] = static_cast<int>(end - given) + over_base;
  }
}

static void check_i32(const at::Tensor& t, const char* name, int64_t dim, int64_t least) {
  APPCORR_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == dim && (t.size(-1) <= 1 || t.stride(-1) == 1), "packed_layout: ", name,
              " must be a CUDA int32 tensor of ", dim, " dimension(s) with unit inner stride");
  APPCORR_CHECK(t.numel() >= least, "packed_layout: ", name, " holds ", t.numel(), " values, ", least, " are needed");
}

void packed_layout_op(const at::Tensor& q_len, const at::Tensor& past, at::Tensor& table, const at::Tensor& free_pages,
                      const at::Tensor& free_start, at::Tensor& q_start, at::Tensor& kv_len, at::Tensor& rows,
                      at::Tensor& req, at::Tensor& pos, at::Tensor& free_next) {
  check_i32(q_len, "q_len", 1, 0);
  const int64_t B = q_len.numel(), N = rows.numel();
  check_i32(past, "past", 1, B);
  check_i32(table, "table", 2, 0);
  check_i32(free_pages, "free_pages", 1, 0);
  check_i32(free_start, "free_start", 1, 1);
  check_i32(q_start, "q_start", 1, B + 1);
  check_i32(kv_len, "kv_len", 1, B);
  check_i32(rows, "rows", 1, 0);
  check_i32(req, "req", 1, N);
  check_i32(pos, "pos", 1, N);
  check_i32(free_next, "free_next", 1, 2);
  APPCORR_CHECK(table.size(0) >= B, "packed_layout: table has ", table.size(0), " rows for ", B, " requests");
  constexpr int64_t kMost = (int64_t(1) << 31) - 2 * kPlThreads;  // a block's next token or request still has a 32-bit number
  APPCORR_CHECK(N < kMost && B < kMost, "packed_layout: too many tokens or requests");
  for (const at::Tensor* t : {&past, (const at::Tensor*)&table, &free_pages, &free_start, (const at::Tensor*)&q_start,
                              (const at::Tensor*)&kv_len, (const at::Tensor*)&rows, (const at::Tensor*)&req,
                              (const at::Tensor*)&pos, (const at::Tensor*)&free_next})
    APPCORR_CHECK(t->device() == q_len.device(), "packed_layout: tensors on different devices");
  // every block reads the inputs while others write the outputs: no output in the place of an input or
  // of another output, as far as they are read and written
  const int64_t W = table.size(1), ld = B > 1 ? table.stride(0) : W;
  APPCORR_CHECK(ld >= W, "packed_layout: the rows of table overlap");
  struct Part {
    const char* name;
    const int *from, *to;
  };
  auto part = [](const char* name, const at::Tensor& t, int64_t n) { return Part{name, t.data_ptr<int>(), t.data_ptr<int>() + n}; };
  const Part in[] = {part("q_len", q_len, B), part("past", past, B), part("free_pages", free_pages, free_pages.numel()),
                     part("free_start", free_start, 1)};
  const Part out[] = {part("q_start", q_start, B + 1), part("kv_len", kv_len, B), part("rows", rows, N),
                      part("req", req, N),             part("pos", pos, N),       part("free_next", free_next, 2)};
  auto meet = [](const Part& a, const Part& b) { return a.from < b.to && b.from < a.to && a.from < a.to && b.from < b.to; };
  auto meets_table = [&](const Part& a) {
    if (a.from == a.to || B == 0 || W == 0) return false;
    const int64_t lo = a.from - table.data_ptr<int>(), hi = lo + (a.to - a.from);
    const int64_t r = lo < W ? 0 : (lo - W) / ld + 1;  // the first row that ends after lo
    return r < B && r * ld < hi;
  };
  for (const Part& a : out) {
    for (const Part& b : in)
      APPCORR_CHECK(!meet(a, b), "packed_layout: ", a.name, " must not lie in the place of ", b.name);
    for (const Part& b : out)
      APPCORR_CHECK(&a == &b || !meet(a, b), "packed_layout: ", a.name, " must not lie in the place of ", b.name);
    APPCORR_CHECK(!meets_table(a), "packed_layout: ", a.name, " must not lie in the place of table");
  }
  for (const Part& b : in) APPCORR_CHECK(!meets_table(b), "packed_layout: table must not lie in the place of ", b.name);
  c10::cuda::CUDAGuard guard(q_len.device());
  LayoutParams p{q_len.data_ptr<int>(), past.data_ptr<int>(), table.data_ptr<int>(), table.stride(0),
                 free_pages.data_ptr<int>(), free_start.data_ptr<int>(), q_start.data_ptr<int>(), kv_len.data_ptr<int>(),
                 rows.data_ptr<int>(), req.data_ptr<int>(), pos.data_ptr<int>(), free_next.data_ptr<int>(),
                 static_cast<int>(B), static_cast<int>(table.size(1)), static_cast<int>(free_pages.numel()),
                 static_cast<int>(N)};
  // one block per 1024 tokens or 32 requests' tables, at most one per SM of a B200
  const int64_t want = std::max((N + kPlThreads - 1) / kPlThreads, (B + 31) / 32);
  const int grid = static_cast<int>(std::min<int64_t>(std::max<int64_t>(want, 1), 148));
  packed_layout_kernel<<<grid, kPlThreads, 0, at::cuda::getCurrentCUDAStream()>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void register_packed_layout_ops(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("packed_layout", &packed_layout_op, py::arg("q_len"), py::arg("past"), py::arg("table"), py::arg("free_pages"),
        py::arg("free_start"), py::arg("q_start"), py::arg("kv_len"), py::arg("rows"), py::arg("req"), py::arg("pos"),
        py::arg("free_next"));
}

}  // namespace appcorr
