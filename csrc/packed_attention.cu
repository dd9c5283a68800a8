// Packed and shared-prefix attention: argument checks, tensor maps and launches (the kernel is in
// packed_attention_sm100.cu).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <cmath>
#include <cudaTypedefs.h>

#include "packed_attention.h"
#include "checks.h"
#include "ops.h"
#include "registry.h"

namespace appcorr {

// [tokens][heads][D] view of the query rows with boxes of `box_tokens` x `box_heads` x 64 columns:
// the query heads of one key head come as consecutive shared-memory rows, token by token.
static CUtensorMap query_tmap(const at::Tensor& q, int64_t heads, int64_t head_dim, int box_heads, int box_tokens) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult r;
    const auto st = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &r);
    TORCH_CHECK(st == cudaSuccess && r == cudaDriverEntryPointSuccess && p != nullptr, "packed attention: cuTensorMapEncodeTiled is unavailable");
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }();
  const int64_t ld = q.size(0) > 1 ? q.stride(0) : heads * head_dim;
  CUtensorMap m;
  cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(q.size(0))};
  cuuint64_t strides[2] = {static_cast<cuuint64_t>(head_dim * 2), static_cast<cuuint64_t>(ld * 2)};
  cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens)};
  cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = encode(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, q.data_ptr(), dims, strides, box, estr,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  APPCORR_CHECK(r == CUDA_SUCCESS, "packed attention: the query tensor map was refused: ", static_cast<int64_t>(r));
  return m;
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
  APPCORR_CHECK(t.is_cuda() && t.scalar_type() == at::kInt && t.dim() == dim && (t.size(-1) <= 1 || t.stride(-1) == 1) && t.numel() >= least,
              "packed attention: ", name, " must be a CUDA int32 tensor of ", dim, " dimension(s), unit inner stride and at least ",
              least, " values");
}

void packed_attention_op(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, at::Tensor& o,
                         const at::Tensor& q_start, const at::Tensor& kv_len, int64_t heads, int64_t kv_heads,
                         int64_t head_dim, double scale, c10::optional<at::Tensor> table, c10::optional<at::Tensor> k_start,
                         c10::optional<at::Tensor> prefix_table, int64_t prefix_len, c10::optional<at::Tensor> lse, const at::Tensor& err) {
  APPCORR_CHECK(head_dim == 64 || head_dim == 128, "packed attention: head_dim must be 64 or 128, got ", head_dim);
  APPCORR_CHECK(heads > 0 && kv_heads > 0 && heads % kv_heads == 0, "packed attention: heads must be a multiple of kv_heads");
  // the running maximum is that of the unscaled products, and what the mask hides is -inf before scaling
  const float scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  APPCORR_CHECK(scale_log2 > 0.f && std::isfinite(scale_log2), "packed attention: scale must be positive and finite in fp32");
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
  APPCORR_CHECK(N < (int64_t(1) << 31) / kPaRows && k.size(0) < (int64_t(1) << 31) - 256, "packed attention: too many rows");
  if (N == 0 || B == 0) return;
  APPCORR_CHECK(k.size(0) > 0, "packed attention: k and v hold no rows");
  c10::cuda::CUDAGuard g(q.device());
  // rows of a tile: tokens x the query heads of one key head. Groups of more than 128 heads are split evenly.
  const int64_t group = heads / kv_heads;
  int64_t parts = (group + 127) / 128;
  while (group % parts) ++parts;
  const int G = static_cast<int>(group / parts), TT = 128 / G;
  const int64_t ldk = k.size(0) > 1 ? k.stride(0) : kv_heads * head_dim, ldv = k.size(0) > 1 ? v.stride(0) : kv_heads * head_dim;
  const CUtensorMap tq = query_tmap(q, heads, head_dim, G, TT), tq1 = query_tmap(q, heads, head_dim, G, 1);
  const CUtensorMap tk = make_tmap_bf16_2d(k.data_ptr(), k.size(0), kv_heads * head_dim, ldk, 128, 64);
  const CUtensorMap tv = make_tmap_bf16_2d(v.data_ptr(), v.size(0), kv_heads * head_dim, ldv, 128, 64);
  PackedAttnParams p{};
  p.B = static_cast<int>(B);
  p.N = static_cast<int>(N);
  p.H = static_cast<int>(heads);
  p.ng = static_cast<int>(parts);
  p.Hv = static_cast<int>(kv_heads * parts);
  p.G = G;
  p.TT = TT;
  p.q_start = q_start.data_ptr<int>();
  p.kv_len = kv_len.data_ptr<int>();
  p.pages = static_cast<int>(k.size(0) / 128);
  p.key_rows = static_cast<int>(k.size(0));
  p.scale_log2 = scale_log2;
  p.o = reinterpret_cast<__nv_bfloat16*>(o.data_ptr());
  p.ldo = o.size(0) > 1 ? o.stride(0) : heads * head_dim;
  p.err = err.data_ptr<int>();
  if (table.has_value()) {
    p.table = table->data_ptr<int>();
    p.ld_table = table->stride(0);
    p.W = static_cast<int>(table->size(1));
  } else {
    p.k_start = k_start->data_ptr<int>();
  }
  p.lse = lse.has_value() ? lse->data_ptr<float>() : nullptr;
  // room for partial results: from the caching allocator, so calls on different streams keep apart
  const int64_t blocks = packed_attention_blocks(), slot_rows = blocks * kPaSlotsPerBlock * kPaRows;
  const int64_t row_words = prefix_len > 0 ? 2 * N * heads * (head_dim + 3) : 0;
  at::Tensor room = at::empty({slot_rows * (head_dim + 2) + blocks * 4 + row_words}, q.options().dtype(at::kFloat));
  p.slots = room.data_ptr<float>();
  p.slot_ml = p.slots + slot_rows * head_dim;
  p.cuts = reinterpret_cast<CutTile*>(p.slot_ml + slot_rows * 2);
  if (prefix_len > 0) {
    p.prefix = prefix_table->data_ptr<int>();
    p.prefix_pages = static_cast<int>(prefix_table->numel());
    p.shared_len = static_cast<int>(prefix_len);
    p.row_o = reinterpret_cast<float*>(p.cuts + blocks);
    p.row_ml = p.row_o + 2 * N * heads * head_dim;
    p.row_parts = reinterpret_cast<int*>(p.row_ml + 4 * N * heads);
  }
  launch_packed_attention(static_cast<int>(head_dim), tq, tq1, tk, tv, p, at::cuda::getCurrentCUDAStream());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void register_packed_attention_ops(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("packed_attention", &packed_attention_op, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("o"), py::arg("q_start"),
        py::arg("kv_len"), py::arg("heads"), py::arg("kv_heads"), py::arg("head_dim"), py::arg("scale"), py::arg("table"),
        py::arg("k_start"), py::arg("prefix_table"), py::arg("prefix_len"), py::arg("lse"),
        py::arg("err"));
}

}  // namespace appcorr
