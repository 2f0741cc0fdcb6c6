"""Refusals of the packed serving operators that need no GPU: the C ABI rejects
what it can see from sizes, strides and alignment before anything is launched
(the pointers below are never read), and the Python ops reject CPU tensors."""
import ctypes

import pytest
import torch

from mka_b200 import _lib, ops

PTR = 0x10000  # a 16-byte aligned address that no call below reads


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        pytest.skip("library not built")
    return _lib.load()


NORM = dict(q=PTR, q_sb=0, q_st=128 * 4, q_sh=128, k=PTR, k_sb=0, k_st=256, k_sh=128, qw=PTR, kw=PTR, w32=0, eps=1e-6,
            cos=PTR, sin=PTR, rsb=0, rst=128, pos=None, p64=0, n_pos=0, qo=PTR, qo_sb=0, qo_st=512, qo_sh=128, ko=PTR,
            ko_sb=0, ko_st=256, ko_sh=128, B=1, T=8, Hq=4, Hkv=2, D=128, stream=None)
VARLEN = dict(q=PTR, q_st=512, q_sh=128, k=PTR, v=PTR, kv_st=256, kv_sh=128, cu_q=PTR, cu_k=PTR, n=2, o=PTR, o_st=512,
              o_sh=128, lse=None, lse_st=1, lse_sh=8, tq=8, tk=8, max_k=8, Hq=4, Hkv=2, D=128, causal=1, scale=0.1,
              ws=None, ws_bytes=0, stream=None)
SHARED = dict(q=PTR, q_sb=512, q_sh=128, kp=PTR, vp=PTR, p_sh=1024, p_st=128, k=PTR, v=PTR, kv_sb=2048, kv_sh=1024,
              kv_st=128, lens=PTR, o=PTR, o_sb=512, o_sh=128, lse=None, lse_sb=4, B=2, Hq=4, Hkv=2, P=8, cap=8, D=128,
              scale=0.1, ws=None, ws_bytes=0, stream=None)


@pytest.mark.parametrize("entry,base,change,code,word", [
    ("fmka_qk_norm_rope_bf16", NORM, dict(q=None), 1, "null"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(ko=None), 1, "null"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(T=0), 1, "empty"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(D=64), 2, "head_dim"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(eps=-1.0), 1, "eps"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(eps=float("nan")), 1, "eps"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(sin=None), 1, "together"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(pos=PTR, n_pos=0), 1, "tables"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(pos=PTR + 4, p64=1, n_pos=9), 1, "aligned"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(q_st=516), 1, "multiples of 8"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(ko_sh=132), 1, "multiples of 8"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(rst=126), 1, "multiples of 4"),
    ("fmka_qk_norm_rope_bf16", NORM, dict(qw=PTR + 8), 1, "16-byte"),
    ("fmka_attn_varlen", VARLEN, dict(n=-1), 1, "negative"),
    ("fmka_attn_varlen", VARLEN, dict(tk=-1), 1, "negative"),
    ("fmka_attn_varlen", VARLEN, dict(cu_k=None), 1, "null"),
    ("fmka_attn_varlen", VARLEN, dict(v=None), 1, "null"),
    ("fmka_attn_varlen", VARLEN, dict(cu_q=PTR + 2), 1, "4-byte"),
    ("fmka_attn_varlen", VARLEN, dict(D=64), 2, "head_dim"),
    ("fmka_attn_varlen", VARLEN, dict(Hq=5), 1, "multiple of kv heads"),
    ("fmka_attn_varlen", VARLEN, dict(Hkv=0), 1, "empty"),
    ("fmka_attn_varlen", VARLEN, dict(scale=float("inf")), 1, "scale"),
    ("fmka_attn_varlen", VARLEN, dict(scale=-0.5), 1, "scale"),
    ("fmka_attn_varlen", VARLEN, dict(kv_st=260), 1, "multiples of 8"),
    ("fmka_attn_varlen", VARLEN, dict(o=PTR + 8), 1, "16-byte"),
    ("fmka_attn_decode_shared", SHARED, dict(B=0), 1, "empty"),
    ("fmka_attn_decode_shared", SHARED, dict(P=-1), 1, "empty"),
    ("fmka_attn_decode_shared", SHARED, dict(kp=None), 1, "null"),
    ("fmka_attn_decode_shared", SHARED, dict(v=None), 1, "null"),
    ("fmka_attn_decode_shared", SHARED, dict(lens=PTR + 1), 1, "4-byte"),
    ("fmka_attn_decode_shared", SHARED, dict(D=256), 2, "head_dim"),
    ("fmka_attn_decode_shared", SHARED, dict(Hq=3), 1, "multiple of kv heads"),
    ("fmka_attn_decode_shared", SHARED, dict(p_st=130), 1, "prefix"),
    ("fmka_attn_decode_shared", SHARED, dict(vp=PTR + 8), 1, "prefix"),
    ("fmka_attn_decode_shared", SHARED, dict(P=5000), 4, "workspace"),
    ("fmka_attn_decode_shared", SHARED, dict(P=5000, ws=PTR, ws_bytes=16), 4, "workspace"),
])
def test_c_abi_refuses(lib, entry, base, change, code, word):
    rc = getattr(lib, entry)(*{**base, **change}.values())
    got, msg = _lib.last_error()
    assert (rc, got) == (code, code)
    assert word in msg


def test_empty_varlen_is_nothing_to_do(lib):
    for change in (dict(n=0), dict(tq=0, q=None, o=None)):
        assert lib.fmka_attn_varlen(*{**VARLEN, **change}.values()) == 0


def test_workspace_sizes_of_bad_shapes_are_zero(lib):
    assert lib.fmka_attn_varlen_workspace_size(0, 8, 8, 4, 2) == 0
    assert lib.fmka_attn_varlen_workspace_size(2, 8, 8, 5, 2) == 0
    assert lib.fmka_attn_decode_shared_workspace_size(0, 4, 2, 8, 8) == 0
    assert lib.fmka_attn_decode_shared_workspace_size(2, 4, 0, 8, 8) == 0


def test_small_problems_need_no_workspace(lib):
    assert lib.fmka_attn_varlen_workspace_size(2, 8, 8, 4, 2) == 0
    assert lib.fmka_attn_decode_shared_workspace_size(2, 4, 2, 8, 8) == 0
    assert lib.fmka_attn_varlen_workspace_size(2, 8, 5000, 4, 2) == 0
    assert lib.fmka_attn_varlen_workspace_size(2, 8, 50000, 4, 2) > 0
    assert lib.fmka_attn_decode_shared_workspace_size(2, 4, 2, 5000, 8) > 0


def test_cpu_tensors_raise():
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.qk_norm_rope(x, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_varlen(x, x, x, cu, cu)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attn_decode_shared(x, x.transpose(0, 1), x.transpose(0, 1), x[:, :, None], x[:, :, None])


def test_strides_of_single_elements_are_ignored():
    t = torch.empty_strided((1, 3, 128), (777, 128, 1))
    assert ops._strides(t) == (0, 128, 1)


@pytest.mark.filterwarnings("ignore:Accessing the data pointer of FakeTensor")
@pytest.mark.parametrize("current", [0, 1])
def test_workspace_size_is_asked_on_the_tensors_device(monkeypatch, current):
    """The size depends on the SMs of the device that the call runs on, not on those of the current one."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    at, calls = [current], []

    class Device:
        def __init__(self, dev):
            self.index = torch.device(dev).index

        def __enter__(self):
            self.before, at[0] = at[0], self.index

        def __exit__(self, *exc):
            at[0] = self.before

    class Lib:
        def __getattr__(self, name):
            def entry(*args):
                calls.append((name, at[0], args))
                return 4096 if name.endswith("workspace_size") else 0
            return entry

    lib = Lib()
    monkeypatch.setattr(ops._lib, "_lib", lib)
    monkeypatch.setattr(ops._lib, "load", lambda: lib)
    monkeypatch.setattr(ops, "_current_device", lambda: at[0])
    monkeypatch.setattr(ops, "_raw_stream", lambda index: 0)
    monkeypatch.setattr(torch.cuda, "device", Device)
    with FakeTensorMode():
        x = torch.empty(4, 2, 128, dtype=torch.bfloat16, device="cuda:1")
        cu = torch.empty(2, dtype=torch.int32, device="cuda:1")
        ops.attn_varlen(x, x, x, cu, cu)
        own = torch.empty(4, 2, 9, 128, dtype=torch.bfloat16, device="cuda:1")
        ops.attn_decode_shared(x, own[0], own[0], own, own)
    assert [(name, dev) for name, dev, _ in calls] == [
        ("fmka_attn_varlen_workspace_size", 1), ("fmka_attn_varlen", 1),
        ("fmka_attn_decode_shared_workspace_size", 1), ("fmka_attn_decode_shared", 1)]
    assert all(args[-2] == 4096 for _, _, args in calls[1::2])
    assert at == [current]


@pytest.mark.parametrize("entry,base", [("fmka_attn_varlen", VARLEN), ("fmka_attn_decode_shared", SHARED)])
@pytest.mark.parametrize("scale", [2.4e38, 3.4e38])
def test_c_abi_refuses_scales_that_overflow_in_base_two(lib, entry, base, scale):
    """The kernels work with scale * log2(e), which has to be finite too: 0 * inf would be NaN."""
    assert getattr(lib, entry)(*{**base, "scale": scale}.values()) == 1
    assert "scale" in _lib.last_error()[1]
