"""Packed-batch operators on host tensors: refused with an exception that says what is wrong."""
import pytest
import torch


def _packed():
    from appcorr_b200.ops import native

    if not native.available():
        pytest.skip("the native extension is not built")
    from appcorr_b200.ops import packed

    return packed


def _i(*s):
    return torch.zeros(*s, dtype=torch.int32)


def test_layout_refuses_host_tensors():
    with pytest.raises(RuntimeError, match="packed_layout: q_len must be a CUDA int32 tensor"):
        _packed().packed_layout(_i(3), _i(3), _i(3, 4), _i(9), _i(1), q_start=_i(4), kv_len=_i(3), rows=_i(5), req=_i(5), pos=_i(5),
                                free_next=_i(2))


def test_rope_refuses_host_tensors_and_head_sizes():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    for dim, text in ((64, "qkv must be a 2-D CUDA bf16"), (80, "head_dim must be 64 or 128, got 80")):
        with pytest.raises(RuntimeError, match=text):
            _packed().qk_norm_rope(b(2, 4 * dim), _i(1, 2), torch.zeros(dim // 2), _i(dim // 2), b(2, 2 * dim), b(2, dim), b(2, dim),
                                   heads=2, kv_heads=1, head_dim=dim)


def test_attention_refuses_host_tensors():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    kw = dict(q_start=_i(2), kv_len=_i(1), heads=2, kv_heads=1, head_dim=64, table=_i(1, 1))
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        _packed().packed_attention(b(1, 128), b(128, 64), b(128, 64), b(1, 128), **kw)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        _packed().shared_prefix_attention(b(1, 128), b(128, 64), b(128, 64), b(1, 128), prefix_table=_i(1), prefix_len=3, **kw)
