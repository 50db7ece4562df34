"""Argument checks of the entry points around an attention layer (CPU: nothing
is launched)."""
import ctypes

import pytest

import esa_native as en

FAKE = 1 << 20  # an aligned address that is never dereferenced


def rotary(mode="fwd", **over):
    a = en.EsaRotaryArgs()
    a.dtype, a.weight_dtype = en.ESA_BF16, en.ESA_BF16
    a.batch, a.num_heads, a.num_kv_heads, a.seq_len = 2, 8, 2, 16
    a.head_dim, a.rotary_dim, a.kv_len, a.eps = 128, 128, 64, 1e-6
    a.inv_freq = a.positions = FAKE
    for name in ("q", "k", "v", "q_out", "k_out", "v_out", "q_grad", "k_grad"):
        setattr(a, name, FAKE)
        for ax, st in zip("bhs", (8 * 16 * 128, 16 * 128, 128)):
            setattr(a, f"{name}_stride_{ax}", st)
    if mode == "bwd":
        a.q_weight_grad = a.k_weight_grad = FAKE
    for name, val in over.items():
        setattr(a, name, val)
    return a


def run_rotary(mode, a, ws=FAKE, ws_bytes=1 << 40):
    lib = en.load()
    if mode == "bwd":
        return lib.esa_qk_norm_rope_bwd(ctypes.byref(a), ws, ws_bytes, None)
    return getattr(lib, "esa_qk_norm_rope_" + mode)(ctypes.byref(a), None)


@pytest.mark.parametrize("mode", ["fwd", "append", "bwd"])
def test_rotary_rejects_bad_arguments(mode):
    bad = [
        (dict(dtype=3), en.ESA_ERR_DTYPE), (dict(weight_dtype=-1), en.ESA_ERR_DTYPE),
        (dict(batch=-1), en.ESA_ERR_SHAPE), (dict(num_heads=0), en.ESA_ERR_SHAPE),
        (dict(num_kv_heads=0), en.ESA_ERR_SHAPE), (dict(seq_len=-1), en.ESA_ERR_SHAPE),
        (dict(rotary_dim=136), en.ESA_ERR_SHAPE), (dict(rotary_dim=0), en.ESA_ERR_SHAPE),
        (dict(interleaved=2), en.ESA_ERR_SHAPE), (dict(eps=-1.0), en.ESA_ERR_SHAPE),
        (dict(eps=float("nan")), en.ESA_ERR_SHAPE),
        (dict(position_stride_b=-16), en.ESA_ERR_SHAPE),
        (dict(batch=1 << 20, seq_len=1 << 20), en.ESA_ERR_SHAPE),
        (dict(head_dim=260), en.ESA_ERR_UNSUPPORTED), (dict(head_dim=130), en.ESA_ERR_UNSUPPORTED),
        (dict(rotary_dim=100), en.ESA_ERR_UNSUPPORTED),
        (dict(q=None), en.ESA_ERR_NULL), (dict(k=None), en.ESA_ERR_NULL),
        (dict(q_out=None), en.ESA_ERR_NULL), (dict(k_out=None), en.ESA_ERR_NULL),
        (dict(inv_freq=None), en.ESA_ERR_NULL), (dict(positions=None), en.ESA_ERR_NULL),
        (dict(q=FAKE + 8), en.ESA_ERR_ALIGN), (dict(k_out_stride_s=132), en.ESA_ERR_ALIGN),
        (dict(q_stride_h=2052), en.ESA_ERR_ALIGN),
    ]
    if mode == "append":
        bad += [(dict(v=None), en.ESA_ERR_NULL), (dict(v_out=None), en.ESA_ERR_NULL),
                (dict(v_out=FAKE + 2), en.ESA_ERR_ALIGN), (dict(kv_len=0), en.ESA_ERR_SHAPE)]
    if mode == "bwd":
        bad += [(dict(q_grad=None), en.ESA_ERR_NULL), (dict(k_grad=FAKE + 4), en.ESA_ERR_ALIGN)]
    for over, status in bad:
        assert run_rotary(mode, rotary(mode, **over)) == status, over
    assert run_rotary(mode, rotary(mode, seq_len=0, q=None)) == en.ESA_OK
    # 8-byte pieces where the halves of the rotation are no whole 16 bytes
    a = rotary(mode, head_dim=72, rotary_dim=72, q=FAKE + 4)
    assert run_rotary(mode, a) == en.ESA_ERR_ALIGN


def test_rotary_workspace():
    lib = en.load()
    n = ctypes.c_size_t()
    a = rotary("bwd")
    assert lib.esa_qk_norm_rope_bwd_workspace_size(ctypes.byref(a), ctypes.byref(n)) == en.ESA_OK
    assert n.value > 0 and n.value % (2 * 128 * 4) == 0
    assert run_rotary("bwd", a, ws_bytes=n.value - 1) == en.ESA_ERR_CAPACITY
    assert run_rotary("bwd", a, ws=None) == en.ESA_ERR_NULL
    assert run_rotary("bwd", a, ws=FAKE + 4) == en.ESA_ERR_ALIGN
    # long batches: no more rows of partial sums than the grid's workgroups
    big = rotary("bwd", batch=64, seq_len=32768)
    lib.esa_qk_norm_rope_bwd_workspace_size(ctypes.byref(big), ctypes.byref(n))
    assert n.value == 1024 * 2 * 128 * 4
    none = rotary("bwd", q_weight_grad=None, k_weight_grad=None)
    lib.esa_qk_norm_rope_bwd_workspace_size(ctypes.byref(none), ctypes.byref(n))
    assert n.value == 0
    assert lib.esa_qk_norm_rope_bwd_workspace_size(None, ctypes.byref(n)) == en.ESA_ERR_NULL
    assert lib.esa_qk_norm_rope_bwd_workspace_size(ctypes.byref(a), None) == en.ESA_ERR_NULL
