"""What ops.linear, ops.window_attention and ops.qkv_cache refuse, before any
device is touched, and the rolling cache's slots."""
import pytest
import torch

import operator_refs as refs
from dfsattn_amd import _lib, ops

BF = torch.bfloat16


def _t(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change", [
    {"x": _t(4, 16, dtype=torch.float32)},
    {"weight": _t(8, 16, dtype=torch.float16)},
    {"weight": _t(8, 15)},
    {"weight": _t(8, 2, 8)},
    {"weight": _t(0, 16)},
    {"x": _t(4, 0), "weight": _t(8, 0)},
    {"bias": _t(7)},
    {"bias": _t(8, dtype=torch.float16)},
    {"bias": _t(8, 1)},
    {"activation": "relu"},
    {"gate": _t(8)},
    {"gate": _t(4, dtype=torch.float32)},
    {"residual": _t(4, 7)},
    {"residual": _t(4, 8, dtype=torch.float32)},
    {"out": _t(5, 8)},
    {"out": _t(4, 8, dtype=torch.float16)},
])
def test_linear_refuses(change):
    args = {"x": _t(4, 16), "weight": _t(8, 16), **change}
    with pytest.raises(ValueError):
        ops.linear(**args)


ATT = dict(q=_t(2, 4, 3, 64), k=_t(2, 2, 9, 64), v=_t(2, 2, 9, 64))


@pytest.mark.parametrize("change", [
    {"q": _t(2, 4, 3, 64, dtype=torch.float32)},
    {"v": _t(2, 2, 9, 64, dtype=torch.float16)},
    {"q": _t(4, 3, 64)},
    {"v": _t(2, 2, 8, 64)},
    {"k": _t(1, 2, 9, 64), "v": _t(1, 2, 9, 64)},
    {"k": _t(2, 3, 9, 64), "v": _t(2, 3, 9, 64)},
    {"q": _t(2, 4, 3, 96), "k": _t(2, 2, 9, 96), "v": _t(2, 2, 9, 96)},
    {"left": -1},
    {"right": -2},
    {"sinks": -1},
    {"q_lens": torch.zeros(2, dtype=torch.int64)},
    {"kv_lens": torch.zeros(3, dtype=torch.int32)},
    {"kv_lens": torch.zeros(4, dtype=torch.int32)[::2]},
    {"rolling": True, "left": 2},
    {"rolling": True, "kv_lens": torch.zeros(2, dtype=torch.int32)},
    {"rolling": True, "left": 5, "sinks": 2, "kv_lens": torch.zeros(2, dtype=torch.int32)},
    {"scale": 0.0},
    {"scale": float("nan")},
])
def test_window_attention_refuses(change):
    with pytest.raises(ValueError):
        ops.window_attention(**{**ATT, **change})


CACHE = dict(q=_t(2, 3, 4, 64), k=_t(2, 3, 2, 64), v=_t(2, 3, 2, 64), k_cache=_t(2, 2, 9, 64), v_cache=_t(2, 2, 9, 64),
             lens=torch.zeros(2, dtype=torch.int32))
SHARED = _t(2, 2, 9, 64)


@pytest.mark.parametrize("change", [
    {"q": _t(2, 3, 4, 64, dtype=torch.float16)},
    {"q": _t(2, 4, 64)},
    {"k": _t(2, 4, 2, 64)},
    {"v": _t(2, 3, 1, 64)},
    {"k_cache": _t(2, 2, 9, 128)},
    {"v_cache": _t(2, 2, 8, 64)},
    {"k_cache": _t(2, 2, 2, 64), "v_cache": _t(2, 2, 2, 64)},
    {"sinks": -1},
    {"sinks": 7, "rolling": True},
    {"k_cache": SHARED, "v_cache": SHARED},
    {"k_cache": _t(2, 1, 9, 64).expand(2, 2, 9, 64)},
    {"k_cache": _t(2, 2, 9, 65)[..., 1:]},
    {"lens": torch.zeros(3, dtype=torch.int32)},
    {"lens": None},
    {"lens": torch.zeros(2)},
    {"new_lens": torch.zeros(1, dtype=torch.int32)},
    {"eps": -1.0},
    {"eps": float("nan")},
    {"q_weight": _t(128)},
    {"k_weight": _t(64, 1)},
    {"table": (torch.zeros(9, 64), torch.zeros(9, 64))},
    {"table": (torch.zeros(9, 32), torch.zeros(8, 32))},
    {"table": (torch.zeros(9, 32, dtype=torch.float64), torch.zeros(9, 32, dtype=torch.float64))},
    {"table": (torch.zeros(9, 32), None)},
])
def test_qkv_cache_refuses(change):
    with pytest.raises(ValueError):
        ops.qkv_cache(**{**CACHE, **change})


def test_head_dims_that_do_not_fit_are_refused():
    for d in (8, 48, 1024):
        with pytest.raises(ValueError):
            ops.qkv_cache(_t(1, 1, 1, d), _t(1, 1, 1, d), _t(1, 1, 1, d), _t(1, 1, 4, d), _t(1, 1, 4, d),
                          torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError):  # more channels than a wave holds
        ops.qkv_cache(_t(1, 1, 65, 128), _t(1, 1, 1, 128), _t(1, 1, 1, 128), _t(1, 1, 4, 128), _t(1, 1, 4, 128),
                      torch.zeros(1, dtype=torch.int32))


def test_operators_refuse_the_cpu_and_gradients():
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.linear(_t(4, 16), _t(8, 16))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.window_attention(**ATT)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.qkv_cache(**CACHE)
    with pytest.raises(RuntimeError, match="no backward"):
        ops.linear(_t(4, 16), _t(8, 16).requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        ops.window_attention(**{**ATT, "v": _t(2, 2, 9, 64).requires_grad_()})
    with pytest.raises(RuntimeError, match="no backward"):
        ops.qkv_cache(**{**CACHE, "q_weight": _t(64).requires_grad_()})


def test_rolling_slots_hold_the_sinks_and_the_newest_tokens():
    for slots, sinks in ((7, 2), (9, 0), (5, 4)):
        held = {}
        for pos in range(40):
            held[refs.slot_of(pos, slots, sinks, True)] = pos
            kept = sorted(held.values())
            ring = slots - sinks
            want = [p for p in range(pos + 1) if p < sinks or p > pos - ring]
            assert kept == want


def test_window_mode_of_full_attention_refuses_what_it_does_not_do():
    from dfsattn_amd.fullattention import full_attention

    q = _t(1, 2, 8, 64)
    for kw in ({"attn_mask": torch.ones(8, 8, dtype=torch.bool)}, {"causal": True}, {"drop_rate": 0.1},
               {"cu_seqlens_q": torch.tensor([0, 5, 8], dtype=torch.int32)}):
        with pytest.raises(NotImplementedError):
            full_attention(q, q, q, mode="window", window=(4, 0), **kw)
    with pytest.raises(ValueError):
        full_attention(q, q, q, mode="window", window=(-4, 0))


def test_window_mode_of_the_processor_leaves_text_modules_dense():
    from dfsattn_amd.replace_wan import Wan_DFSAttn_Processor2_0

    args = ("window", 0.3, 16, 128, None, 0, [], 12, 12, 0.0, True)
    assert Wan_DFSAttn_Processor2_0(*args, False, window=(4, 4), sinks=2).branch() == "window"
    assert Wan_DFSAttn_Processor2_0(*args, True).branch() == "dense"


def test_operators_refuse_gradients_of_what_they_write():
    with pytest.raises(RuntimeError, match="no backward"):
        ops.linear(_t(4, 16), _t(8, 16), out=_t(4, 8).requires_grad_())
    with pytest.raises(RuntimeError, match="no backward"):
        ops.window_attention(**ATT, out=_t(2, 4, 3, 64).requires_grad_())
    for name in ("k_cache", "v_cache"):
        with pytest.raises(RuntimeError, match="no backward"):
            ops.qkv_cache(**{**CACHE, name: _t(2, 2, 9, 64).requires_grad_()})


def test_limits_behind_every_length_are_kept_within_their_type():
    for n in (1 << 40, 1 << 63, 1 << 64, 10 ** 30):
        assert ops._limit("window_attention", "left", n) == 1 << 40
    assert ops._limit("window_attention", "left", None) == -1
    with pytest.raises(ValueError):  # more sinks than the cache has slots
        ops.window_attention(**{**ATT, "rolling": True, "left": 0, "sinks": 1 << 64,
                                "kv_lens": torch.zeros(2, dtype=torch.int32)})


def test_sizes_beyond_a_launch_are_refused():
    """The library's own checks, which end a call before its launch."""
    def linear(rows, n, k):
        a = _lib.LinearArgs()
        a.rows, a.n, a.k, a.x_stride, a.w_stride, a.out_stride = rows, n, k, k, k, n
        a.x = a.w = a.out = a.workspace = 16
        a.workspace_bytes = max(_lib.lib().dfs_linear_workspace_size(rows, n, k, 1), 0)
        _lib.call("dfs_linear", bytes(a), None)

    with pytest.raises(_lib.DfsKernelError, match="2\\^21"):
        linear(1, 8, 1 << 21)
    with pytest.raises(_lib.DfsKernelError, match="too many outputs"):
        linear(1 << 20, 1 << 20, 64)
    with pytest.raises(_lib.DfsKernelError, match="too many outputs"):
        linear(1, 1 << 28, 8)
    a = _lib.CacheArgs()
    a.batch, a.tokens, a.q_heads, a.kv_heads, a.head_dim, a.slots = 1 << 6, 1 << 20, 1, 1, 16, 1 << 20
    for name in ("q", "k", "v", "q_out", "k_cache", "v_cache", "lens"):
        setattr(a, name, 16)
    with pytest.raises(_lib.DfsKernelError, match="sizes too large"):
        _lib.call("dfs_qkv_cache", bytes(a), None)
    a = _lib.WindowArgs()
    a.batch, a.q_heads, a.kv_heads, a.q_rows, a.slots, a.head_dim = 1 << 13, 1 << 13, 1 << 13, 1, 8, 64
    a.left = a.right = -1
    a.scale = 0.125
    for name in ("q", "k", "v", "out"):
        setattr(a, name, 16)
    with pytest.raises(_lib.DfsKernelError, match="too many rows"):
        _lib.call("dfs_window_attention", bytes(a), None)


# --------------------------------------------------------------------------
# channels that share an element
# --------------------------------------------------------------------------

def _shared_channels(*shape):
    """Tensors of this shape whose channels (and more axes) have stride 0."""
    whole = torch.arange(4096, dtype=BF).repeat(8)[:torch.Size(shape).numel()].reshape(shape)
    return [whole[..., :1].expand(shape), whole[..., 8:9].expand(shape), torch.tensor(3.0, dtype=BF).expand(shape),
            whole[:1, ..., :1].expand(shape), whole[:, :, :1, :1].expand(shape)]


def test_channels_that_share_an_element_are_copied():
    """The kernels read a row's channels one behind the other: rows whose
    channels are one element are never read in place."""
    for t in _shared_channels(2, 2, 9, 64):
        assert t.stride(3) == 0
        assert not ops._chunk_rows(t.shape, t.stride()) and not ops._own_rows(t.shape, t.stride())
        c = ops._in_chunks(t)
        assert c.is_contiguous() and torch.equal(c, t)
        for name in ("q", "k", "v"):
            x = {**{n: (2, 2, 9, 64) for n in "qkv"}}
            strides = {n: (1152, 576, 64, 1) for n in "qkv"}
            strides[name] = t.stride()
            plan = ops._window_plan(x["q"], strides["q"], x["k"], strides["k"], x["v"], strides["v"], (BF, BF, BF),
                                    None, None, 0, 0, False, False, None)
            assert not plan[3] and plan[2][-1] == 1  # not in place; out has channels of its own
            shapes = (*x.values(), (2, 9, 9, 64), (2, 9, 9, 64))
            dense = ops._contiguous_stride((2, 9, 9, 64))
            assert not ops._cache_plan(shapes, (*strides.values(), dense, dense), (BF,) * 5, (None, None), None, 1e-6,
                                       0, False)[1]
    for shape, stride in (((2, 2, 9, 64), (1152, 576, 64, 1)), ((2, 2, 9, 64), (0, 0, 64, 1)),
                          ((1, 1, 1, 64), (5, 3, 7, 1)), ((4, 1), (8, 5))):
        assert ops._chunk_rows(shape, stride)


def test_window_mode_refuses_other_operands_than_its_inputs():
    """mode "window" multiplies in q's dtype: another operand_dtype is refused,
    not passed over."""
    from dfsattn_amd.fullattention import full_attention

    for dtype, other in ((BF, torch.float16), (torch.float16, BF)):
        q = _t(1, 2, 8, 64, dtype=dtype)
        with pytest.raises(ValueError, match="operand_dtype"):
            full_attention(q, q, q, mode="window", window=(4, 0), operand_dtype=other)
        for same in (dtype, None):  # as far as the device
            with pytest.raises(RuntimeError, match="ROCm GPU"):
                full_attention(q, q, q, mode="window", window=(4, 0), operand_dtype=same)


# --------------------------------------------------------------------------
# rows that are written share no memory
# --------------------------------------------------------------------------

def test_rows_to_write_that_overlap_each_other_are_refused():
    buf = torch.zeros(200000, dtype=BF)
    shape = (2, 2, 9, 64)
    good = [(1152, 576, 64, 1), (1152, 64, 128, 1), (64, 128, 256, 1), (9216, 4608, 512, 1), (1168, 584, 64, 1)]
    bad = [(1152, 576, 32, 1), (1152, 64, 64, 1), (1152, 512, 64, 1), (576, 576, 64, 1), (8, 576, 64, 1)]
    for stride in good + bad:
        view = buf.as_strided(shape, stride)
        cells = torch.arange(200000).as_strided(shape, stride).flatten()
        assert (cells.unique().numel() == cells.numel()) == (stride in good)
        cache = {**CACHE, "k_cache": view}
        with pytest.raises(RuntimeError if stride in good else ValueError,
                           match="ROCm GPU" if stride in good else "rows of their own"):
            ops.qkv_cache(**cache)
        q = _t(*shape)
        with pytest.raises(RuntimeError if stride in good else ValueError,
                           match="ROCm GPU" if stride in good else "rows of its own"):
            ops.window_attention(q, q, q, out=view)


def test_caches_that_overlap_each_other_are_refused():
    """Their rows may alternate in one tensor, but no element may be both's."""
    shape = (2, 2, 9, 64)
    buf = torch.zeros(100000, dtype=BF)
    cells = torch.arange(100000)
    rng = torch.Generator().manual_seed(0)
    orders = [(2304, 1152, 128, 1), (2304, 128, 256, 1), (1152, 576, 64, 1), (4608, 64, 256, 1)]
    shifts = [0, 8, 64, 128, 512, 576, 1152, 1216, 2304, 2368, 4608, 20000]
    shifts += (torch.randint(0, 1200, (40,), generator=rng) * 8).tolist()
    kinds = {True: 0, False: 0}
    for stride in orders:
        for shift in shifts:
            for first, second in ((0, shift), (shift, 0)):
                k, v = (buf.as_strided(shape, stride, at) for at in (first, second))
                at = [cells.as_strided(shape, stride, o).flatten() for o in (first, second)]
                shared = torch.cat(at).unique().numel() < 2 * at[0].numel()
                kinds[shared] += 1
                with pytest.raises(ValueError if shared else RuntimeError, match="same memory" if shared else "ROCm GPU"):
                    ops.qkv_cache(**{**CACHE, "k_cache": k, "v_cache": v})
    assert min(kinds.values()) > 50
    # other strides than k's: apart, or refused
    k = buf.as_strided(shape, orders[0])
    with pytest.raises(ValueError, match="same memory"):
        ops.qkv_cache(**{**CACHE, "k_cache": k, "v_cache": buf.as_strided(shape, orders[1], 64)})
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.qkv_cache(**{**CACHE, "k_cache": k, "v_cache": buf.as_strided(shape, orders[1], 50000)})


def test_scales_that_single_precision_cannot_hold_are_refused():
    """Below 1e-45 a scale is 0 in fp32, and 0 times a hidden key's minus
    infinity would be NaN."""
    for scale in (1e-31, 1e-46, 5e-324, 1e30, float("inf"), -0.125):
        with pytest.raises(ValueError, match="scale"):
            ops.window_attention(**ATT, scale=scale)
        a = _lib.WindowArgs()
        a.batch = a.q_heads = a.kv_heads = a.q_rows = a.slots = 1
        a.head_dim, a.left, a.right, a.scale = 64, -1, -1, scale
        for name in ("q", "k", "v", "out"):
            setattr(a, name, 16)
        with pytest.raises(_lib.DfsKernelError, match="scale"):
            _lib.call("dfs_window_attention", bytes(a), None)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.window_attention(**ATT, scale=1e-30)


def test_window_mode_of_the_processor_passes_its_operand_dtype_on(monkeypatch):
    """The operand_dtype that is set for the dense path is not dropped in mode
    "window": it is refused where it is not the inputs' dtype."""
    from dfsattn_amd import replace_wan
    from dfsattn_amd.dit import DiTAttention

    attn = DiTAttention(128, 2, 1e-6, device="cpu", dtype=BF)
    attn.set_processor(replace_wan.Wan_DFSAttn_Processor2_0("window", 0.3, 16, 128, None, 0, [], 12, 12, 0.0, True, False,
                                                            window=(4, 4)))
    x = _t(1, 8, 128)
    for dtype, error in ((torch.float16, ValueError), (BF, RuntimeError), (None, RuntimeError)):
        monkeypatch.setattr(replace_wan.WanDFSAttention, "operand_dtype", dtype)
        with pytest.raises(error, match="operand_dtype" if error is ValueError else "ROCm GPU"), torch.no_grad():
            attn(x)
