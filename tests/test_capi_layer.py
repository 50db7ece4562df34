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


def window(**over):
    w = en.EsaWindow()
    w.window, w.sinks = 64, 4
    for name, val in over.items():
        setattr(w, name, val)
    return w


def sink_args(cls, **over):
    a = cls()
    a.dtype = en.ESA_BF16
    a.batch, a.num_heads, a.num_kv_heads = 2, 8, 2
    a.q_len, a.kv_len, a.head_dim, a.sm_scale = 300, 300, 64, 0.125
    names = ("q", "k", "v", "o") if cls is en.EsaFwdArgs else \
        ("q", "k", "v", "o", "dout", "dq", "dk", "dv")
    for name in names:
        setattr(a, name, FAKE)
        for ax, st in zip("bhs", (8 * 300 * 64, 300 * 64, 64)):
            setattr(a, f"{name}_stride_{ax}", st)
    a.lse, a.lse_stride_b, a.lse_stride_h = FAKE, 8 * 300, 300
    for name, val in over.items():
        setattr(a, name, val)
    return a


@pytest.mark.parametrize("cls", [en.EsaFwdArgs, en.EsaBwdArgs])
def test_sink_window_rejects_bad_arguments(cls):
    lib = en.load()
    fwd = cls is en.EsaFwdArgs
    run = lib.esa_sink_window_fwd if fwd else lib.esa_sink_window_bwd
    size = lib.esa_sink_window_fwd_workspace_size if fwd else \
        lib.esa_sink_window_bwd_workspace_size

    def call(a, w, ws=FAKE, n=1 << 50):
        return run(ctypes.byref(a), None if w is None else ctypes.byref(w), ws, n, None)

    big = (1 << 31) // 256
    shape = [
        (dict(dtype=9), {}, en.ESA_ERR_DTYPE), (dict(batch=-1), {}, en.ESA_ERR_SHAPE),
        (dict(num_heads=7), {}, en.ESA_ERR_SHAPE), (dict(kv_len=0), {}, en.ESA_ERR_SHAPE),
        (dict(q_len=301), {}, en.ESA_ERR_SHAPE), (dict(q_len=-1), {}, en.ESA_ERR_SHAPE),
        (dict(kv_len=(1 << 26) + 1), {}, en.ESA_ERR_SHAPE),
        ({}, dict(window=0), en.ESA_ERR_SHAPE), ({}, dict(sinks=-1), en.ESA_ERR_SHAPE),
        ({}, dict(position_stride_b=-1), en.ESA_ERR_SHAPE),
        (dict(head_dim=136), {}, en.ESA_ERR_UNSUPPORTED),
        (dict(head_dim=20), {}, en.ESA_ERR_UNSUPPORTED),
        (dict(dtype=en.ESA_F32, head_dim=130), {}, en.ESA_ERR_UNSUPPORTED),
        (dict(sm_scale=0.0), {}, en.ESA_ERR_UNSUPPORTED),
        (dict(sm_scale=float("inf")), {}, en.ESA_ERR_UNSUPPORTED),
        (dict(batch=1 << 22, num_heads=8), {}, en.ESA_ERR_SHAPE),
    ]
    n = ctypes.c_size_t()
    for over, wover, status in shape:
        a, w = sink_args(cls, **over), window(**wover)
        assert call(a, w) == status, (over, wover)
        assert size(ctypes.byref(a), ctypes.byref(w), ctypes.byref(n)) == status, (over, wover)
    memory = [(dict(q=None), en.ESA_ERR_NULL), (dict(o=None), en.ESA_ERR_NULL),
              (dict(k=FAKE + 8), en.ESA_ERR_ALIGN), (dict(v_stride_s=68), en.ESA_ERR_ALIGN),
              (dict(o_stride_h=4), en.ESA_ERR_ALIGN), (dict(k_stride_s=big), en.ESA_ERR_UNSUPPORTED),
              (dict(v_stride_s=-64), en.ESA_ERR_UNSUPPORTED)]
    if not fwd:
        memory += [(dict(dout=None), en.ESA_ERR_NULL), (dict(lse=None), en.ESA_ERR_NULL),
                   (dict(dk=FAKE + 2), en.ESA_ERR_ALIGN), (dict(dq_stride_s=65), en.ESA_ERR_ALIGN),
                   (dict(q_stride_s=big), en.ESA_ERR_UNSUPPORTED),
                   (dict(dout_stride_s=big), en.ESA_ERR_UNSUPPORTED)]
    for over, status in memory:
        assert call(sink_args(cls, **over), window()) == status, over
    assert call(sink_args(cls), None) == en.ESA_ERR_NULL
    assert size(ctypes.byref(sink_args(cls)), ctypes.byref(window()), None) == en.ESA_ERR_NULL
    # no rows: nothing is read
    assert call(sink_args(cls, q_len=0, q=None), window()) == en.ESA_OK
    assert call(sink_args(cls, batch=0, q=None), window()) == en.ESA_OK
    # a window past the cache is one over the whole cache; sinks then add nothing
    a = sink_args(cls)
    sizes = []
    for w in (window(window=300, sinks=0), window(window=2 ** 31 - 1, sinks=2 ** 31 - 1)):
        assert size(ctypes.byref(a), ctypes.byref(w), ctypes.byref(n)) == en.ESA_OK
        sizes.append(n.value)
    assert sizes[0] == sizes[1]


def test_sink_window_workspaces():
    lib = en.load()
    n = ctypes.c_size_t()
    # a prefill needs none; a decode step's key ranges one part each
    a = sink_args(en.EsaFwdArgs)
    assert lib.esa_sink_window_fwd_workspace_size(ctypes.byref(a), ctypes.byref(window()),
                                                  ctypes.byref(n)) == en.ESA_OK
    assert n.value == 0
    a = sink_args(en.EsaFwdArgs, q_len=1, kv_len=4000)
    w = window(window=3000)
    lib.esa_sink_window_fwd_workspace_size(ctypes.byref(a), ctypes.byref(w), ctypes.byref(n))
    need = n.value
    assert need > 0 and need % (2 * 2 * 16 * 67 * 4) == 0
    run = lambda ws, size: lib.esa_sink_window_fwd(ctypes.byref(a), ctypes.byref(w), ws, size, None)
    assert run(None, need) == en.ESA_ERR_NULL
    assert run(FAKE + 4, need) == en.ESA_ERR_ALIGN
    assert run(FAKE, need - 1) == en.ESA_ERR_CAPACITY
    # the backward: two floats a row, and the parts of the sinks' blocks, which
    # stay bounded however many sinks there are
    b = sink_args(en.EsaBwdArgs)
    lib.esa_sink_window_bwd_workspace_size(ctypes.byref(b), ctypes.byref(window(sinks=0)),
                                           ctypes.byref(n))
    rows = 2 * 8 * 300 * 4
    assert n.value >= 2 * rows
    lib.esa_sink_window_bwd_workspace_size(ctypes.byref(b), ctypes.byref(window()),
                                           ctypes.byref(n))
    need = n.value
    assert need > 2 * rows
    assert lib.esa_sink_window_bwd(ctypes.byref(b), ctypes.byref(window()), FAKE, need - 1,
                                   None) == en.ESA_ERR_CAPACITY
    assert lib.esa_sink_window_bwd(ctypes.byref(b), ctypes.byref(window()), None, need,
                                   None) == en.ESA_ERR_NULL
    long = sink_args(en.EsaBwdArgs, q_len=1 << 20, kv_len=1 << 20, head_dim=128)
    lib.esa_sink_window_bwd_workspace_size(ctypes.byref(long),
                                           ctypes.byref(window(sinks=1 << 19)), ctypes.byref(n))
    assert n.value < 2 * 2 * 8 * (1 << 20) * 4 + (4 << 30)
