// Causal grouped-query attention over a packed batch: request b's new tokens are the rows
// q_start[b] .. q_start[b + 1] of q, its keys the kv_len[b] rows of its cache pages (or of the packed
// K / V rows from k_start[b]), the new tokens' own keys last:
//   o_t = sum_j p_tj v_j / sum_j p_tj,   p_tj = exp(scale q_t . k_j - max_j),   j <= kv_len - q_len + t
// A shared prefix of P keys (its own page list) stands in front of every request's keys and is
// visible to every token. A row that sees no key is zero and its log-sum-exp is -inf.
//
// One warp per (token, head): the definition, one key at a time.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "sm100_common.cuh"
#include "checks.h"
#include "registry.h"

namespace appcorr {

using bf16 = __nv_bfloat16;

struct PaParams {
  const bf16* q;
  const bf16* k;
  const bf16* v;
  bf16* o;
  long ldq, ldk, ldv, ldo, kv_rows;
  const int* q_start;
  const int* kv_len;
  const int* table;
  long ld_table;
  int W;
  const int* k_start;
  const int* prefix;
  int prefix_len;
  float* lse;  // [N, H]
  float scale;
  int B, N, H, Hkv;
};

template <int D>
__global__ void packed_attention_simple(PaParams p) {
  const int n = blockIdx.x, h = blockIdx.y * blockDim.y + threadIdx.y, lane = threadIdx.x;
  if (h >= p.H || n >= p.q_start[p.B]) return;
  int lo = 0, hi = p.B;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.q_start[mid] <= n) lo = mid;
    else hi = mid;
  }
  constexpr int E = D / 32;
  const int b = lo, kvh = h / (p.H / p.Hkv);
  float q[E], acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(p.q[n * p.ldq + h * D + lane * E + e]) * p.scale;
    acc[e] = 0.f;
  }
  float m = -INFINITY, l = 0.f;
  const int own = max(p.kv_len[b] - p.q_start[b + 1] + n + 1, 0);  // own keys this token sees
  for (int j = -p.prefix_len; j < own; ++j) {
    long row;
    if (j < 0 || p.table != nullptr) {
      const int i = j < 0 ? j + p.prefix_len : j, blk = i >> 7;
      const int page = j < 0 ? p.prefix[blk] : (blk < p.W ? p.table[b * p.ld_table + blk] : -1);
      row = page < 0 ? -1 : (long)page * 128 + (i & 127);
    } else {
      row = (long)p.k_start[b] + j;
    }
    const bool have = row >= 0 && row < p.kv_rows;
    float s = 0.f, vv[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      s += have ? q[e] * __bfloat162float(p.k[row * p.ldk + kvh * D + lane * E + e]) : 0.f;
      vv[e] = have ? __bfloat162float(p.v[row * p.ldv + kvh * D + lane * E + e]) : 0.f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const float mn = fmaxf(m, s), c = mn == -INFINITY ? 1.f : expf(m - mn), w = mn == -INFINITY ? 0.f : expf(s - mn);
    m = mn;
    l = l * c + w;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * c + w * vv[e];
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < E; ++e) p.o[n * p.ldo + h * D + lane * E + e] = __float2bfloat16_rn(acc[e] * inv);
  if (p.lse != nullptr && lane == 0) p.lse[(long)n * p.H + h] = m + logf(l);
}

static void pa_check_rows(const at::Tensor& t, const char* name, int64_t width) {
  APPCORR_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1, "packed attention: ", name,
              " must be a 2-D CUDA bf16 tensor with unit inner stride");
  APPCORR_CHECK(t.size(1) == width, "packed attention: ", name, " rows hold ", t.size(1), " values, ", width, " are needed");
  APPCORR_CHECK((t.size(0) <= 1 || (t.stride(0) % 8 == 0 && t.stride(0) >= width)) &&
                  (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
              "packed attention: ", name, " rows must be 16-byte aligned and must not overlap");
}
static void pa_check_i32(const at::Tensor& t, const char* name, int64_t dim, int64_t least) {
  APPCORR_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == dim && t.stride(-1) == 1 && t.numel() >= least,
              "packed attention: ", name, " must be a CUDA int32 tensor of ", dim, " dimension(s), unit inner stride and at least ",
              least, " values");
}

void packed_attention_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& o,
                         const at::Tensor& q_start, const at::Tensor& kv_len, int64_t heads, int64_t kv_heads,
                         int64_t head_dim, double scale, c10::optional<at::Tensor> table, c10::optional<at::Tensor> k_start,
                         c10::optional<at::Tensor> prefix_table, int64_t prefix_len, c10::optional<at::Tensor> lse) {
  APPCORR_CHECK(head_dim == 64 || head_dim == 128, "packed attention: head_dim must be 64 or 128, got ", head_dim);
  APPCORR_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "packed attention: heads must be a multiple of kv_heads");
  pa_check_rows(q, "q", heads * head_dim);
  pa_check_rows(o, "o", heads * head_dim);
  pa_check_rows(k, "k", kv_heads * head_dim);
  pa_check_rows(v, "v", kv_heads * head_dim);
  const int64_t N = q.size(0), B = kv_len.numel();
  pa_check_i32(kv_len, "kv_len", 1, 0);
  pa_check_i32(q_start, "q_start", 1, B + 1);
  APPCORR_CHECK(o.size(0) >= N, "packed attention: o has ", o.size(0), " rows for ", N, " tokens");
  APPCORR_CHECK(k.size(0) == v.size(0), "packed attention: k and v have different numbers of rows");
  APPCORR_CHECK(table.has_value() != k_start.has_value(), "packed attention: give either table (cache pages) or k_start (packed rows)");
  if (table.has_value()) {
    pa_check_i32(*table, "table", 2, 0);
    APPCORR_CHECK(table->size(0) >= B, "packed attention: table has ", table->size(0), " rows for ", B, " requests");
    APPCORR_CHECK(k.size(0) % 128 == 0, "packed attention: a page pool has a multiple of 128 rows");
  } else {
    pa_check_i32(*k_start, "k_start", 1, B);
  }
  APPCORR_CHECK(prefix_len >= 0 && prefix_len < (int64_t(1) << 30), "packed attention: prefix_len out of range");
  if (prefix_len > 0) {
    APPCORR_CHECK(prefix_table.has_value(), "packed attention: a shared prefix needs its page list");
    pa_check_i32(*prefix_table, "prefix_table", 1, (prefix_len + 127) / 128);
    APPCORR_CHECK(k.size(0) % 128 == 0, "packed attention: a page pool has a multiple of 128 rows");
  }
  if (lse.has_value()) {
    APPCORR_CHECK(lse->is_cuda() && lse->scalar_type() == at::kFloat && lse->is_contiguous() && lse->numel() >= N * heads,
                "packed attention: lse must be contiguous CUDA fp32 [tokens, heads]");
  }
  for (const at::Tensor* t : {&k, &v, (const at::Tensor*)&o, &q_start, &kv_len})
    APPCORR_CHECK(t->device() == q.device(), "packed attention: tensors on different devices");
  for (auto* t : {&table, &k_start, &prefix_table, &lse})
    APPCORR_CHECK(!t->has_value() || (*t)->device() == q.device(), "packed attention: tensors on different devices");
  if (N == 0 || B == 0) return;
  c10::cuda::CUDAGuard guard(q.device());
  PaParams p{reinterpret_cast<const bf16*>(q.data_ptr()), reinterpret_cast<const bf16*>(k.data_ptr()),
             reinterpret_cast<const bf16*>(v.data_ptr()), reinterpret_cast<bf16*>(o.data_ptr()), q.stride(0), k.stride(0),
             v.stride(0), o.stride(0), k.size(0), q_start.data_ptr<int>(), kv_len.data_ptr<int>(),
             table.has_value() ? table->data_ptr<int>() : nullptr, table.has_value() ? table->stride(0) : 0,
             table.has_value() ? static_cast<int>(table->size(1)) : 0, k_start.has_value() ? k_start->data_ptr<int>() : nullptr,
             prefix_len > 0 ? prefix_table->data_ptr<int>() : nullptr, static_cast<int>(prefix_len),
             lse.has_value() ? lse->data_ptr<float>() : nullptr, static_cast<float>(scale), static_cast<int>(B),
             static_cast<int>(N), static_cast<int>(heads), static_cast<int>(kv_heads)};
  dim3 grid(static_cast<unsigned>(N), static_cast<unsigned>((heads + 3) / 4));
  auto st = at::cuda::getCurrentCUDAStream();
  if (head_dim == 128) packed_attention_simple<128><<<grid, dim3(32, 4), 0, st>>>(p);
  else packed_attention_simple<64><<<grid, dim3(32, 4), 0, st>>>(p);
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void register_packed_attention_ops(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("packed_attention", &packed_attention_op, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("q_start"),
        py::arg("kv_len"), py::arg("heads"), py::arg("kv_heads"), py::arg("head_dim"), py::arg("scale"), py::arg("table"),
        py::arg("k_start"), py::arg("prefix_table"), py::arg("prefix_len"), py::arg("lse"));
}

}  // namespace appcorr
