"""What the operators around a block refuse, before any launch (on the CPU)."""
import ctypes

import pytest
import torch

import pack3d_amd as p3d
from pack3d_amd import _lib
from pack3d_amd.dropout import mask_args, threshold_of


def test_struct_mirrors_match_c_sizes():
    out = (ctypes.c_int64 * 4)()
    assert _lib.lib().p3d_block_struct_sizes(out) == 0
    assert list(out) == [ctypes.sizeof(s) for s in (_lib.Dropout, _lib.NormArgs, _lib.BlockArgs, _lib.RotaryArgs)]


def test_no_cpu_fallback():
    x = torch.zeros(1, 4, 8)
    for call in (lambda: p3d.block_norm(x, p3d.Norm()), lambda: p3d.block_residual(x, x),
                 lambda: p3d.counter_dropout(x, 0.1, 1),
                 lambda: p3d.apply_rotary(x[None], torch.arange(4), p3d.rotary_frequencies(4)[0])):
        with pytest.raises(ValueError, match="HIP device"):
            call()


@pytest.mark.parametrize("p", [-0.1, 1.0, 1.5, float("nan")])
def test_rates(p):
    with pytest.raises(ValueError, match="rate"):
        threshold_of(p)


def test_thresholds():
    assert [threshold_of(p) for p in (0.0, 2.0 ** -18, 2.0 ** -16, 0.1, 0.5, 1 - 2.0 ** -20)] == [0, 0, 1, 6554, 32768, 65535]


@pytest.mark.parametrize("seed", [None, -1, 2 ** 63, (1,), (1, -1), 1.5, "a", torch.zeros(2), torch.zeros(3, dtype=torch.int64)])
def test_seeds(seed):
    with pytest.raises(ValueError, match="seed"):
        mask_args(0.1, seed, torch.device("cpu"))


def _block_args(**kw):
    a = _lib.BlockArgs()
    a.tokens, a.samples, a.splits, a.grid, a.dim = 4, 2, 1, 2, 64
    a.x = a.y = a.out = 16
    a.x_stride = a.y_stride = 64
    a.alpha = 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,message", [
    ({"dim": 0}, "dim"), ({"dim": 8193}, "dim"), ({"tokens": 0}, "row count"), ({"tokens": 2 ** 31}, "row count"),
    ({"samples": 2 ** 30}, "row count"), ({"splits": 5}, "splits"), ({"splits": 0}, "splits"), ({"grid": 3}, "grid"),
    ({"outer": 3}, "dtype"), ({"outer": 1, "inner": 2}, "16-bit stream"), ({"outer": 1, "inner": 0}, "16-bit stream"),
    ({"x": None}, "null pointer"), ({"gate_kind": 4}, "gate kind"), ({"gate_kind": 1}, "disagree"), ({"gate": 16}, "disagree"),
    ({"y": None}, "nothing to compute"), ({"y": None, "scale": 16}, "without y"), ({"y": None, "alpha": 2.0}, "without y"),
    ({"out": None}, "null output"), ({"post": _lib.NormArgs(None, None, 3, 0.0)}, "norm kind"),
    ({"next": _lib.NormArgs(None, None, 1, 0.0)}, "null output"),
    ({"x_stride": 2 ** 29}, "strides"), ({"y_stride": -1}, "strides"),
    ({"dropout": _lib.Dropout(None, 0, 0, 65536, 0)}, "threshold"), ({"dropout": _lib.Dropout(None, 0, 0, -1, 0)}, "threshold"),
])
def test_block_entry_points_refuse(change, message):
    with pytest.raises(RuntimeError, match=message):
        _lib.call("p3d_block_fwd", _block_args(**change), None)
    if message not in ("null output",):
        with pytest.raises(RuntimeError, match=message):
            _lib.call("p3d_block_bwd", _block_args(dout=16, **change), None)


@pytest.mark.parametrize("change,message", [
    ({}, "upstream"), ({"dn": 16}, "upstream"), ({"dout": 16, "dn": 16}, "next norm"),
    ({"dout": 16, "post": _lib.NormArgs(None, None, 1, 0.0)}, "statistics"),
    ({"dout": 16}, "null output"), ({"dout": 16, "dy": 16, "dgate": 16}, "dgate without"),
    ({"dout": 16, "dy": 16, "gate": 16, "gate_kind": 2}, "null output"),
    ({"dout": 16, "dy": 16, "gate": 16, "gate_kind": 1, "dgate": 16}, "work"),
    ({"dout": 16, "dy": 16, "d_param": (ctypes.c_void_p * 5)(16)}, "d_param without"),
    ({"dout": 16, "dy": 16, "d_param": (ctypes.c_void_p * 5)(None, None, 16), "scale": 16}, "work"),
    ({"dout": 16, "dy": 16, "d_param": (ctypes.c_void_p * 5)(None, None, None, 16),
      "next": _lib.NormArgs(16, None, 1, 0.0)}, "d_param without"),
    ({"y": None, "out": None, "next": _lib.NormArgs(None, None, 1, 0.0)}, "upstream"),
    ({"y": None, "out": None, "dn": 16, "stats": 16, "next": _lib.NormArgs(None, None, 1, 0.0)}, "null output"),
])
def test_block_backward_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        _lib.call("p3d_block_bwd", _block_args(**change), None)
    with pytest.raises(RuntimeError, match="null args"):
        _lib.call("p3d_block_bwd", None, None)


def test_dropout_entry_point_refuses():
    d = _lib.Dropout(None, 1, 0, 100, 0)
    for args, message in (((None, 16, 8, 0, d), "null"), ((16, 16, 0, 0, d), "count"), ((16, 16, 8, 3, d), "dtype"),
                          ((16, 16, 8, 0, None), "null"), ((16, 16, 2 ** 50, 0, d), "count"),
                          ((16, 16, 8, 0, _lib.Dropout(None, 1, 0, 65536, 0)), "threshold")):
        with pytest.raises(RuntimeError, match=message):
            _lib.call("p3d_dropout_apply", *args, None)


def _rotary_args(**kw):
    a = _lib.RotaryArgs()
    a.x[0] = a.y[0] = _lib.View(16, 64, 64, 64)
    a.heads[0] = 4
    a.tokens, a.count, a.batch, a.head_dim, a.pairs, a.axes = 4, 1, 1, 64, 32, 1
    a.axis_pairs[0] = 32
    a.positions = a.freqs = 16
    a.magnitude = 1.0
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("change,message", [
    ({"count": 0}, "tensors"), ({"count": 5}, "tensors"), ({"dtype": 3}, "dtype"), ({"batch": 0}, "sizes"), ({"tokens": 0}, "sizes"),
    ({"head_dim": 1025}, "sizes"), ({"pairs": 0}, "pairs"), ({"pairs": 33}, "pairs"), ({"positions": None}, "null"),
    ({"freqs": None}, "null"), ({"axes": 0}, "axes"), ({"axes": 4}, "axes"), ({"pairs": 31}, "add up"), ({"count": 2}, "null tensor"),
])
def test_rotary_entry_point_refuses(change, message):
    with pytest.raises(RuntimeError, match=message):
        _lib.call("p3d_rotary", _rotary_args(**change), None)


def test_rotary_entry_point_refuses_heads():
    a = _rotary_args()
    a.heads[0] = 5000
    with pytest.raises(RuntimeError, match="too large"):
        _lib.call("p3d_rotary", a, None)


@pytest.mark.parametrize("kw", [{"pairs": 0}, {"pairs": (1, 2, 3, 4)}, {"pairs": (-1, 3)}, {"pairs": 4, "scaling": "other"},
                                {"pairs": 4, "factor": 0.5}, {"pairs": 4, "base": 1.0}, {"pairs": 4, "scaling": "parts"},
                                {"pairs": 4, "scaling": "parts", "trained": 8, "fast": 1.0}])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        p3d.rotary_frequencies(kw.pop("pairs"), **kw)


@pytest.mark.parametrize("kw", [{"layout": "other"}, {"fraction": 0.0}, {"fraction": 1.5}, {"scaling": "parts"}, {"factor": 0.1}])
def test_encoding_refusals(kw):
    with pytest.raises(ValueError):
        p3d.RotaryEncoding(**kw)


@pytest.mark.parametrize("samples,tokens", [(1, 1), (1, 7), (3, 4913), (5000, 1), (1, 2 ** 31 - 1), (100000, 3)])
@pytest.mark.parametrize("dim", [1, 5, 64, 192, 512, 513, 8192])
@pytest.mark.parametrize("round_", [0, 1, 256, 768, 2048])
def test_splits_stay_within_what_the_kernels_take(samples, tokens, dim, round_):
    splits, grid = _lib.ops().block_split(samples, tokens, dim, round_)
    assert 1 <= splits <= tokens and 1 <= grid <= splits * samples and splits * samples < 2 ** 31
