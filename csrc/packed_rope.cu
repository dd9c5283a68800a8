// Norms of queries and keys per head, the rotation over several position axes and the K / V write
// into cache rows, in one pass over the packed projection rows [q heads | k heads | v heads].
//
//   y = x * rsqrt(mean(x^2) + eps) * w                       (each head of D; skipped where w is not given)
//   (y_i, y_{i + D/2}) -> (y_i cos t_i - y_{i + D/2} sin t_i, y_{i + D/2} cos t_i + y_i sin t_i)
//   t_i = pos[axis_i, token] * inv_freq_i
//
// The angle is reduced in turns before any rounding matters: inv_freq / 2 pi is formed as a pair of
// floats (product and its fma residual), multiplied by the integer position the same way, and only
// the fraction of a turn goes to sincospif. Positions below 2^24 keep full fp32 accuracy; an angle
// formed in one fp32 product would be off by 1e-3 rad at position 30000.
//
// Bound: HBM, every projected value read once and written once (20011 tokens of 48 heads x 64: 246 MB in
// 46.7 us = 5.3 TB/s, 0.82 of a plain copy). At 1 to 2 waves of blocks it is the latency of a load, sines,
// store chain: 1424 tokens of 36 heads x 128, 26 MB, take 7.5 us without norms and 8.3 with them where the
// inputs come from HBM, 5.1 and 6.2 where L2 still holds them; 61 of them with norms 2.7 us.
// A lane holds 8 values of a head's first half and the 8 they are paired with, so both loads and
// stores are 16 bytes and the rotation needs no exchange; a head is D / 16 lanes (the norm is 3 or
// 2 shuffles) and a warp walks its token's heads 32 / (D / 16) at a time with the next ones' loads
// in flight. A token's sines are computed once per warp, split over its lane groups and exchanged
// by shuffles. One warp serves a token when there are enough of them, up to 8 when there are few (see
// the launch).
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include "sm100_common.cuh"
#include "checks.h"
#include "registry.h"

namespace appcorr {

struct RopeParams {
  const __nv_bfloat16* qkv;
  long ld;
  const int* pos;  // [axes, ld_pos]
  long ld_pos;
  const float* inv_freq;
  const int* axis;
  int axes;
  const int* rows;  // cache row of each token (nullptr: the token itself; < 0: not written)
  long cache_rows;
  const __nv_bfloat16* qw;
  const __nv_bfloat16* kw;
  float eps;
  __nv_bfloat16* q_out;
  long ld_q;
  __nv_bfloat16* k;
  __nv_bfloat16* v;
  long ld_k, ld_v;
  int N, H, Hkv;
};

constexpr int kRopeThreads = 256;

__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16x2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}

// WPT: warps per token
template <int D, int WPT>
__global__ void __launch_bounds__(kRopeThreads) qk_norm_rope_kernel(RopeParams p) {
  constexpr int LPH = D / 16;      // lanes per head
  constexpr int HPW = 32 / LPH;    // heads a warp holds at a time
  constexpr int PPG = 8 / HPW;     // of a lane's 8 pairs, those its group computes the sines of
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = lane % LPH, g = lane / LPH;
  const long tok = (long)blockIdx.x * (kRopeThreads / 32 / WPT) + warp / WPT;
  if (tok >= p.N) return;
  const int heads = p.H + 2 * p.Hkv;
  const __nv_bfloat16* src = p.qkv + tok * p.ld + c * 8;
  const int h0 = (warp % WPT) * HPW + g;
  uint4 a = make_uint4(0, 0, 0, 0), b = a;
  if (h0 < heads) {
    a = *reinterpret_cast<const uint4*>(src + (long)h0 * D);
    b = *reinterpret_cast<const uint4*>(src + (long)h0 * D + D / 2);
  }
  const long row = p.rows ? (long)p.rows[tok] : tok;
  float sn[8], cs[8];
  {
    float s[PPG], co[PPG];
#pragma unroll
    for (int j = 0; j < PPG; ++j) {
      const int i = c * 8 + g * PPG + j;
      const float f = p.inv_freq[i];
      const int ax = p.axis[i];
      const float x = (unsigned)ax < (unsigned)p.axes ? (float)p.pos[ax * p.ld_pos + tok] : 0.f;
      constexpr double kInv2Pi = 0.15915494309189533577;
      constexpr float kHi = (float)kInv2Pi, kLo = (float)(kInv2Pi - (double)kHi);
      const float hi = f * kHi, lo = fmaf(f, kLo, fmaf(f, kHi, -hi));  // inv_freq / 2 pi
      const float t = x * hi, e = fmaf(x, lo, fmaf(x, hi, -t));        // turns
      sincospif(2.f * ((t - rintf(t)) + e), &s[j], &co[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int from = (j / PPG) * LPH + c;
      sn[j] = __shfl_sync(0xffffffffu, s[j % PPG], from);
      cs[j] = __shfl_sync(0xffffffffu, co[j % PPG], from);
    }
  }
  const bool keep = row >= 0 && row < p.cache_rows;
  for (int base = (warp % WPT) * HPW; base < heads; base += WPT * HPW) {
    const int h = base + g, hn = h + WPT * HPW;
    uint4 na = make_uint4(0, 0, 0, 0), nb = na;
    if (hn < heads) {
      na = *reinterpret_cast<const uint4*>(src + (long)hn * D);
      nb = *reinterpret_cast<const uint4*>(src + (long)hn * D + D / 2);
    }
    const bool isq = h < p.H, isv = h >= p.H + p.Hkv;
    __nv_bfloat16* dst = isq ? p.q_out + tok * p.ld_q + (long)h * D
                         : isv ? p.v + row * p.ld_v + (long)(h - p.H - p.Hkv) * D
                               : p.k + row * p.ld_k + (long)(h - p.H) * D;
    float x[8], y[8];
    unpack8(a, x);
    unpack8(b, y);
    const __nv_bfloat16* w = isq ? p.qw : isv ? nullptr : p.kw;
    float ss = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w != nullptr) {
      const float r = rsqrtf(ss * (1.f / D) + p.eps);
      float wx[8], wy[8];
      unpack8(*reinterpret_cast<const uint4*>(w + c * 8), wx);
      unpack8(*reinterpret_cast<const uint4*>(w + c * 8 + D / 2), wy);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] *= r * wx[j];
        y[j] *= r * wy[j];
      }
    }
    if (!isv) {
      float u[8], v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = x[j] * cs[j] - y[j] * sn[j];
        v[j] = y[j] * cs[j] + x[j] * sn[j];
      }
      a = pack8(u);
      b = pack8(v);
    }
    if (h < heads && (isq || keep)) {
      *reinterpret_cast<uint4*>(dst + c * 8) = a;
      *reinterpret_cast<uint4*>(dst + c * 8 + D / 2) = b;
    }
    a = na;
    b = nb;
  }
}

static void check_rows_bf16(const at::Tensor& t, const char* name, int64_t width) {
  APPCORR_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.stride(1) == 1, "qk_norm_rope: ", name,
              " must be a 2-D CUDA bf16 tensor with unit inner stride");
  APPCORR_CHECK(t.size(1) == width, "qk_norm_rope: ", name, " rows hold ", t.size(1), " values, ", width, " are needed");
  APPCORR_CHECK((t.size(0) <= 1 || t.stride(0) % 8 == 0) && (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0,
              "qk_norm_rope: ", name, " rows must be 16-byte aligned");
}
static void check_written_rows(const at::Tensor& t, const char* name, int64_t width) {
  check_rows_bf16(t, name, width);
  APPCORR_CHECK(t.size(0) <= 1 || t.stride(0) >= width, "qk_norm_rope: ", name, " rows must not overlap");
}

void qk_norm_rope_op(const at::Tensor& qkv, const at::Tensor& pos, const at::Tensor& inv_freq, const at::Tensor& axis,
                     at::Tensor& q_out, at::Tensor& k_cache, at::Tensor& v_cache, int64_t heads, int64_t kv_heads,
                     int64_t head_dim, c10::optional<at::Tensor> rows, c10::optional<at::Tensor> q_weight,
                     c10::optional<at::Tensor> k_weight, double eps) {
  APPCORR_CHECK(head_dim == 64 || head_dim == 128, "qk_norm_rope: head_dim must be 64 or 128, got ", head_dim);
  APPCORR_CHECK(heads > 0 && kv_heads > 0, "qk_norm_rope: heads and kv_heads must be positive");
  check_rows_bf16(qkv, "qkv", (heads + 2 * kv_heads) * head_dim);
  check_written_rows(q_out, "q_out", heads * head_dim);
  check_written_rows(k_cache, "k_cache", kv_heads * head_dim);
  check_written_rows(v_cache, "v_cache", kv_heads * head_dim);
  const int64_t N = qkv.size(0);
  APPCORR_CHECK(N < (int64_t(1) << 31), "qk_norm_rope: too many tokens");
  APPCORR_CHECK(q_out.size(0) >= N, "qk_norm_rope: q_out has ", q_out.size(0), " rows for ", N, " tokens");
  APPCORR_CHECK(pos.is_cuda() && pos.scalar_type() == at::kInt && pos.dim() == 2 && pos.size(1) == N &&
                  (N <= 1 || pos.stride(1) == 1), "qk_norm_rope: pos must be CUDA int32 [axes, tokens]");
  APPCORR_CHECK(inv_freq.is_cuda() && inv_freq.scalar_type() == at::kFloat && inv_freq.is_contiguous() &&
                  inv_freq.numel() == head_dim / 2, "qk_norm_rope: inv_freq must be CUDA fp32 [head_dim / 2]");
  APPCORR_CHECK(axis.is_cuda() && axis.scalar_type() == at::kInt && axis.is_contiguous() && axis.numel() == head_dim / 2,
              "qk_norm_rope: axis must be CUDA int32 [head_dim / 2]");
  if (rows.has_value()) {
    APPCORR_CHECK(rows->is_cuda() && rows->scalar_type() == at::kInt && rows->is_contiguous() && rows->numel() == N,
                "qk_norm_rope: rows must be contiguous CUDA int32 [tokens]");
  } else {
    APPCORR_CHECK(k_cache.size(0) >= N && v_cache.size(0) >= N, "qk_norm_rope: without rows the caches need a row per token");
  }
  for (auto* w : {&q_weight, &k_weight})
    if (w->has_value()) {
      APPCORR_CHECK((*w)->is_cuda() && (*w)->scalar_type() == at::kBFloat16 && (*w)->is_contiguous() &&
                      (*w)->numel() == head_dim && (reinterpret_cast<uintptr_t>((*w)->data_ptr()) & 15) == 0,
                  "qk_norm_rope: norm weights must be aligned CUDA bf16 [head_dim]");
    }
  for (const at::Tensor* t : {&pos, &inv_freq, &axis, (const at::Tensor*)&q_out, (const at::Tensor*)&k_cache,
                              (const at::Tensor*)&v_cache})
    APPCORR_CHECK(t->device() == qkv.device(), "qk_norm_rope: tensors on different devices");
  for (auto* t : {&rows, &q_weight, &k_weight})
    APPCORR_CHECK(!t->has_value() || (*t)->device() == qkv.device(), "qk_norm_rope: tensors on different devices");
  if (N == 0) return;
  c10::cuda::CUDAGuard guard(qkv.device());
  using bf = __nv_bfloat16;
  RopeParams p{reinterpret_cast<const bf*>(qkv.data_ptr()), qkv.stride(0), pos.data_ptr<int>(), pos.stride(0),
               inv_freq.data_ptr<float>(), axis.data_ptr<int>(), static_cast<int>(pos.size(0)),
               rows.has_value() ? rows->data_ptr<int>() : nullptr, std::min(k_cache.size(0), v_cache.size(0)),
               q_weight.has_value() ? reinterpret_cast<const bf*>(q_weight->data_ptr()) : nullptr,
               k_weight.has_value() ? reinterpret_cast<const bf*>(k_weight->data_ptr()) : nullptr, static_cast<float>(eps),
               reinterpret_cast<bf*>(q_out.data_ptr()), q_out.stride(0), reinterpret_cast<bf*>(k_cache.data_ptr()),
               reinterpret_cast<bf*>(v_cache.data_ptr()), k_cache.stride(0), v_cache.stride(0), static_cast<int>(N),
               static_cast<int>(heads), static_cast<int>(kv_heads)};
  auto st = at::cuda::getCurrentCUDAStream();
  // Warps per token: fewer repeat the sines less, more shorten the chain of a single token. Measured in us
  // at 1 / 2 / 4 / 8 with 36 heads x 128 and norms, inputs from HBM (from L2): 61 tokens 5.9 / 4.2 / 3.5 / 2.8
  // (5.1 / 3.9 / 3.1 / 2.6), 600: 8.7 / 6.6 / 5.5 / 6.3 (5.4 / 4.6 / 4.2 / 4.7), 1424: 10.2 / 8.3 / 9.3 / 10.7
  // (7.2 / 6.2 / 6.3 / 8.1), 3000: 13.0 / 13.9 / 15.3 / 18.4, 20011: 67 / 70 / 79 / 104.
  const int wpt = N >= 2048 ? 1 : (N >= 1024 ? 2 : (N >= 512 ? 4 : 8));
  auto go = [&](auto kern) {
    const long per = kRopeThreads / 32 / wpt;
    kern<<<static_cast<unsigned>((N + per - 1) / per), kRopeThreads, 0, st>>>(p);
  };
  if (head_dim == 128) {
    if (wpt == 1) go(qk_norm_rope_kernel<128, 1>);
    else if (wpt == 2) go(qk_norm_rope_kernel<128, 2>);
    else if (wpt == 4) go(qk_norm_rope_kernel<128, 4>);
    else go(qk_norm_rope_kernel<128, 8>);
  } else {
    if (wpt == 1) go(qk_norm_rope_kernel<64, 1>);
    else if (wpt == 2) go(qk_norm_rope_kernel<64, 2>);
    else if (wpt == 4) go(qk_norm_rope_kernel<64, 4>);
    else go(qk_norm_rope_kernel<64, 8>);
  }
  C10_CUDA_KERNEL_LAUNCH_CHECK();
}

void register_packed_rope_ops(pybind11::module_& m) {
  namespace py = pybind11;
  m.def("qk_norm_rope", &qk_norm_rope_op, py::arg("qkv"), py::arg("pos"), py::arg("inv_freq"), py::arg("axis"),
        py::arg("q_out"), py::arg("k_cache"), py::arg("v_cache"), py::arg("heads"), py::arg("kv_heads"), py::arg("head_dim"),
        py::arg("rows"), py::arg("q_weight"), py::arg("k_weight"), py::arg("eps"));
}

}  // namespace appcorr
