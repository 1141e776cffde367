"""What the operators between a step's products and after them refuse, without a GPU: the Python
calls' checks and the entry points' own; and their launches at sizes that no test could run."""

from __future__ import annotations

import ctypes
import math
from pathlib import Path

import pytest
import torch

from test_host_sanitize import _run, driver  # noqa: F401  (a fixture)
from test_operator_launches import _launches
from verification.computation import operators as ops

LIB = Path(__file__).resolve().parents[1] / "pots-2.0_amd" / "libpots_mi355x.so"
E_ARG = -4
F32, BF16, E4M3, INT8 = 0, 1, 2, 3
NAMES = ("rms_norm_forward", "rms_norm_quantized", "rms_norm_backward", "rotary_turn",
         "gated_silu_forward", "gated_silu_backward", "gradient_norm", "clip_gradients", "sgd_step")


@pytest.fixture(scope="module")
def abi():
    if not LIB.exists():
        pytest.fail(f"{LIB} is not built")
    lib = ctypes.CDLL(str(LIB))
    for name in NAMES:
        getattr(lib, f"pots_{name}").restype = ctypes.c_int
    for name in ("rms_norm_backward", "gradient_norm", "clip_gradients", "sgd_step"):
        getattr(lib, f"pots_{name}_work").restype = ctypes.c_uint64
    return lib


def _t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


X, W = _t(3, 8), _t(8)
H, BF, I64 = torch.float16, torch.bfloat16, torch.int64


@pytest.mark.parametrize("x, w, kw, message", [
    (_t(3, 8, dtype=H), W, {}, "float32 or bfloat16"), (X, _t(8, dtype=H), {}, "float32 or bfloat16"),
    (X, _t(7), {}, "weight"), (X, _t(1, 8), {}, "weight"), (_t(3, 0), _t(0), {}, "dim"),
    (_t(), W, {}, "dim"), (_t(1, ops.MAX_NORM_DIM + 1), _t(ops.MAX_NORM_DIM + 1), {}, "dim"),
    (X, W, {"residual": _t(2, 8)}, "residual"),
    (X, W, {"residual": _t(3, 8, dtype=H)}, "float32 or bfloat16"),
    (X, W, {"eps": 0.0}, "eps"), (X, W, {"eps": -1e-6}, "eps"), (X, W, {"eps": math.nan}, "eps"),
    (X, W, {"eps": math.inf}, "eps"), (X, W, {"eps": 1e39}, "eps"), (X, W, {"eps": 1e-39}, "eps"), (X, W, {}, "GPU"),
])
def test_norms_refuse(x, w, kw, message):
    for call in (ops.rms_norm_forward, ops.rms_norm_quantized, ops.rms_norm):
        with pytest.raises(ValueError, match=message):
            call(x, w, **kw)


def test_norm_types_and_blocks_are_refused():
    with pytest.raises(ValueError, match="out_dtype"):
        ops.rms_norm_forward(X, W, out_dtype=H)
    with pytest.raises(ValueError, match="dtype"):
        ops.rms_norm_quantized(X, W, dtype=torch.float8_e5m2)
    for block in (0, 16, 48, 512, -32):
        with pytest.raises(ValueError, match="block"):
            ops.rms_norm_quantized(X, W, block=block)


@pytest.mark.parametrize("dy, total, w, rstd, kw, message", [
    (_t(3, 9), X, W, _t(3), {}, "dy"), (_t(3, 8, dtype=H), X, W, _t(3), {}, "float32 or bfloat16"),
    (X, X, _t(9), _t(3), {}, "weight"), (X, X, W, _t(4), {}, "rstd"),
    (X, X, W, _t(3, dtype=BF), {}, "rstd"), (X, X, W, _t(3), {"dtotal": _t(3, 8, dtype=BF)}, "dtotal"),
    (X, X, W, _t(3), {"dtotal": _t(2, 8)}, "dtotal"), (X, X, W, _t(3), {"x_dtype": H}, "x_dtype"),
    (X, X, W, _t(3), {}, "GPU"),
])
def test_norm_backward_refuses(dy, total, w, rstd, kw, message):
    with pytest.raises(ValueError, match=message):
        ops.rms_norm_backward(dy, total, w, rstd, **kw)


Q, K, AT, F = _t(2, 4, 5, 8), _t(2, 2, 5, 8), torch.arange(5), _t(4)


@pytest.mark.parametrize("q, k, at, f, kw, message", [
    (Q[0], K, AT, F, {}, "batch"), (Q, K[0], AT, F, {}, "batch"), (Q.to(H), K.to(H), AT, F, {}, "float32"),
    (Q, K.to(BF), AT, F, {}, "k must"), (Q, K[:, :, :4], AT, F, {}, "k has"),
    (Q[:, :0], K, AT, F, {}, "heads"), (Q, K[:, :0], AT, F, {}, "heads"),
    (Q, K, AT.float(), F, {}, "positions"), (Q, K, AT[:4], F, {}, "positions"),
    (Q, K, AT.expand(3, 5), F, {}, "positions"), (Q, K, AT.expand(2, 2, 5), F, {}, "positions"),
    (Q, K, torch.tensor(3), F, {}, "positions"), (Q, K, AT, _t(5), {}, "frequencies"),
    (Q, K, AT, _t(0), {}, "frequencies"), (Q, K, AT, F.to(H), {}, "frequencies"),
    (Q, K, AT, F[None], {}, "frequencies"), (Q, K, AT.expand(2, 5), F, {"sections": (1, 2)}, "sections"),
    (Q, K, AT.expand(2, 5), F, {"sections": (5, -1)}, "sections"),
    (Q, K, AT.expand(5, 5), F, {"sections": (1, 1, 1, 1, 0)}, "sections"),
    (Q, K, AT.expand(3, 5), F, {"sections": (2, 2)}, "positions"),
    (Q, K, AT, F, {"sections": (4,)}, "positions"), (Q, K, AT.expand(1, 5), F, {"sections": ()}, "sections"),
    (_t(1, 1, 5, 1025), _t(1, 1, 5, 1025), AT, F, {}, "head_dim"), (Q, K, AT, F, {}, "GPU"),
])
def test_rotary_refuses(q, k, at, f, kw, message):
    for call in (ops.rotary_forward, ops.rotary_backward, ops.rotary):
        with pytest.raises(ValueError, match=message):
            call(q, k, at, f, **kw)


def test_rotary_frequencies():
    f = ops.rotary_frequencies(8, base=100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1, 100**-.25, .1, 100**-.75],
                                                                       dtype=torch.float64))
    for width in (0, 7, -2):
        with pytest.raises(ValueError, match="width"):
            ops.rotary_frequencies(width, device="cpu")


@pytest.mark.parametrize("gate, up, message", [
    (X.to(H), X.to(H), "float32 or bfloat16"), (X, X.to(BF), "up must"), (X, _t(3, 9), "up has"),
    (_t(), _t(), "columns"), (X, X, "GPU")])
def test_gated_silu_refuses(gate, up, message):
    for call in (lambda: ops.gated_silu_forward(gate, up), lambda: ops.gated_silu(gate, up),
                 lambda: ops.gated_silu_backward(gate, gate, up)):
        with pytest.raises(ValueError, match=message):
            call()
    with pytest.raises(ValueError, match="dout"):
        ops.gated_silu_backward(_t(2, 8), X, X)


@pytest.mark.parametrize("gradients, message", [
    ([], "at least one"), ([X, None], "tensors"), ([X, X.to(H)], "dense"),
    ([X, X.to_sparse()], "dense"), ([X], "GPU")])
def test_gradient_lists_refuse(gradients, message):
    for call in (lambda: ops.gradient_norm(gradients), lambda: ops.clip_gradients(gradients, 1.0),
                 lambda: ops.sgd_step(gradients, gradients, 0.1)):
        with pytest.raises(ValueError, match=message):
            call()


def test_updates_refuse():
    for bad in (0.0, -1.0, math.nan, 1e-50):
        with pytest.raises(ValueError, match="max_norm"):
            ops.clip_gradients([X], bad)
        with pytest.raises(ValueError, match="max_norm"):
            ops.sgd_step([X], [X], 0.1, max_norm=bad)
    for bad in (math.nan, math.inf, 1e39):
        with pytest.raises(ValueError, match="eta"):
            ops.sgd_step([X], [X], bad)
    with pytest.raises(ValueError, match="shapes"):
        ops.sgd_step([X, X], [X], 0.1)
    with pytest.raises(ValueError, match="shapes"):
        ops.sgd_step([X], [_t(8, 3)], 0.1)
    for out in ([], [_t(8, 3)], [X.to(BF)], [X, X]):
        with pytest.raises(ValueError, match="out"):
            ops.clip_gradients([X], 1.0, out=out)
        with pytest.raises(ValueError, match="out"):
            ops.sgd_step([X], [X], 0.1, out=out)
    for t in (_t(8, 3).t(), _t(1, 8).expand(3, 8)):
        with pytest.raises(ValueError, match="contiguous"):
            ops.clip_gradients([t], 1.0)
        with pytest.raises(ValueError, match="contiguous"):
            ops.sgd_step([X], [X], 1.0, out=[t])


# ---- the entry points' own checks -----------------------------------------------------------

def _norm(**kw):
    a = dict(rows=3, dim=8, block=0, x=0, total=0, weight=0, y=0, eps=1e-6)
    a.update(kw)
    return ops._NORM.pack(*(0,) * 12, *(8,) * 5, a["rows"], a["dim"], a["block"], a["x"], a["total"],
                          a["weight"], a["y"], a["eps"])


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=(1 << 14) + 1), dict(rows=1 << 31), dict(x=2),
                                dict(total=2), dict(weight=4), dict(eps=0.0), dict(eps=1e-39), dict(eps=-1.0),
                                dict(eps=math.nan), dict(eps=math.inf), {}])
def test_norm_entry_points_refuse(abi, kw):
    """Sizes, types and numbers out of range; with none, null pointers."""
    assert abi.pots_rms_norm_forward(_norm(**kw), None) == E_ARG
    assert abi.pots_rms_norm_backward(_norm(**kw), None, None) == E_ARG
    for y in (E4M3, INT8):
        assert abi.pots_rms_norm_quantized(_norm(**{"y": y, **kw}), None) == E_ARG


def test_norm_entry_points_refuse_types_and_blocks(abi):
    assert abi.pots_rms_norm_forward(_norm(y=E4M3, rows=0), None) == E_ARG
    assert abi.pots_rms_norm_backward(_norm(y=INT8, rows=0), None, None) == E_ARG
    for kw in (dict(y=F32), dict(y=BF16), dict(y=4), dict(y=E4M3, block=16), dict(y=INT8, block=512)):
        assert abi.pots_rms_norm_quantized(_norm(rows=0, **kw), None) == E_ARG
    assert abi.pots_rms_norm_quantized(_norm(rows=0, y=E4M3, block=64), None) == 0
    assert abi.pots_rms_norm_forward(_norm(rows=0), None) == 0
    assert abi.pots_rms_norm_backward(_norm(rows=0), None, None) == 0  # dweight is null
    assert abi.pots_rms_norm_backward_work(_norm()) == 0


def _rotary(**kw):
    a = dict(b=1, h=2, kv=1, n=3, d=8, pairs=4, axes=1, ends=(4, 4, 4, 4), dtype=0, f=0, bits=64)
    a.update(kw)
    return ops._ROTARY.pack(*(0,) * 21, a["b"], a["h"], a["kv"], a["n"], a["d"], a["pairs"], a["axes"],
                            *a["ends"], a["dtype"], a["f"], a["bits"], 0, 0)


@pytest.mark.parametrize("kw", [dict(h=0), dict(kv=0), dict(d=0), dict(d=1025), dict(pairs=0),
                                dict(pairs=5), dict(axes=0), dict(axes=5), dict(dtype=2), dict(f=1),
                                dict(bits=16), dict(ends=(3, 4, 4, 4)), dict(h=65537),
                                dict(axes=2, ends=(5, 4, 4, 4)), dict(axes=2, ends=(2, 3, 4, 4)),
                                dict(b=1 << 16, n=1 << 15), dict(pairs=1 << 31), {}])
def test_rotary_entry_point_refuses(abi, kw):
    assert abi.pots_rotary_turn(_rotary(**kw), None) == E_ARG


def _gated(rows=3, columns=8, dtype=0):
    return ops._GATED.pack(*(0,) * 6, 8, 8, 8, rows, columns, dtype)


@pytest.mark.parametrize("kw", [dict(dtype=2), dict(columns=(1 << 30) + 1),
                                dict(rows=1 << 20, columns=(1 << 20) + 1), {}])
def test_gated_entry_points_refuse(abi, kw):
    assert abi.pots_gated_silu_forward(_gated(**kw), None) == E_ARG
    assert abi.pots_gated_silu_backward(_gated(**kw), None) == E_ARG


def _gradients(entries, max_norm=1.0, eta=0.1, norm=1 << 40, count=None):
    return ops._GRADIENTS.pack(norm, max_norm, eta, len(entries) if count is None else count, 0) + \
        b"".join(ops._GRADIENT.pack(*e) for e in entries)


A, B, C = 1 << 41, 1 << 42, 1 << 43  # addresses; nothing reads them


@pytest.mark.parametrize("block", [
    _gradients([]), _gradients([], count=65537), _gradients([(A, B, C, 8, 2, 0)]),
    _gradients([(A, B, C, 8, 0, 0)], norm=0), _gradients([(0, B, C, 8, 0, 0)]),
    _gradients([(A, B, C, (1 << 42) + 1, 0, 0)]), _gradients([(A, B, C, 1 << 42, 0, 0)] * 3),
    _gradients([(A, B, C, 8, 0, 0)])])  # the last: no scratch
def test_gradient_entry_points_refuse(abi, block):
    for name in ("gradient_norm", "clip_gradients", "sgd_step"):
        assert getattr(abi, f"pots_{name}")(block, None, None) == E_ARG


@pytest.mark.parametrize("block", [
    _gradients([(A, B, C, 8, 0, 0)], max_norm=0.0), _gradients([(A, B, C, 8, 0, 0)], max_norm=math.nan),
    _gradients([(A, B, 0, 8, 0, 0)]),
    _gradients([(A, B, C, 8, 0, 0), (A + 64, B + 64, C + 31, 8, 0, 0)]),   # two outs overlap
    _gradients([(A, B, A + 4, 8, 0, 0)]),                                  # shifted over its own
    _gradients([(A, B, A + 32, 8, 0, 0), (A + 32, B, C, 8, 0, 0)]),        # over another input
    _gradients([(A, B, C, 100, 0, 0), (A + 400, B, A + 396, 8, 0, 0)])])
def test_updates_that_would_overwrite_are_refused(abi, block):
    scratch = ctypes.c_void_p(C + (1 << 20))
    assert abi.pots_clip_gradients(block, scratch, None) == E_ARG
    assert abi.pots_sgd_step(block, scratch, None) == E_ARG


def test_steps_have_checks_of_their_own(abi):
    scratch = ctypes.c_void_p(C + (1 << 20))
    for block in (_gradients([(A, 0, C, 8, 0, 0)]), _gradients([(A, B, C, 8, 0, 2)]),
                  _gradients([(A, B, C, 8, 0, 0)], eta=math.inf),
                  _gradients([(A, B, B + 4, 8, 0, 0)]), _gradients([(A, B, A, 8, 0, 1)])):
        assert abi.pots_sgd_step(block, scratch, None) == E_ARG


def test_null_blocks(abi):
    for name in NAMES:
        fn = getattr(abi, f"pots_{name}")
        args = (None, None, None) if hasattr(abi, f"pots_{name}_work") else (None, None)
        assert fn(*args) == E_ARG
    for name in ("rms_norm_backward", "gradient_norm", "clip_gradients", "sgd_step"):
        assert getattr(abi, f"pots_{name}_work")(None) == 0


# ---- launches -------------------------------------------------------------------------------

@pytest.mark.parametrize("rows", [1, 5, 100000, (1 << 31) - 1])
@pytest.mark.parametrize("dim", [1, 256, 1000, 1536, 2048, 4096, 8192, 1 << 14])
def test_norms_of_any_rows_are_one_launch(driver, rows, dim):  # noqa: F811
    got = _launches(driver, f"rms_norm_forward,{rows},{dim},0,{BF16},{F32},{F32},{BF16}",
                    f"rms_norm_quantized,{rows},{dim},128,{F32},{F32},{F32},{INT8}",
                    f"rms_norm_backward,{rows},{dim},0,{BF16},{F32},{F32},{BF16}")
    assert [rc for rc, _, _ in got] == [0, 0, 0]
    assert [len(x) for _, _, x in got] == [1, 1, 2]
    assert got[2][1] == 4 * dim * got[2][2][0][1] and got[2][2][1][0] == "norm_join"


@pytest.mark.parametrize("n, d, pairs", [((1 << 31) - 1, 2, 1), ((1 << 31) - 1, 1024, 512),
                                         (1, 64, 32), (8192, 128, 64), (100, 20, 5)])
def test_turns_of_any_tokens(driver, n, d, pairs):  # noqa: F811
    """A block's angles fit its LDS, and every token has one."""
    (rc, _, launches), = _launches(driver, f"rotary_turn,1,3,1,{n},{d},{pairs},{BF16}")
    blocks = sum(x for _, x, _ in launches)
    per = -(-n // blocks)
    assert rc == 0 and per * pairs <= 1024 and per <= 64 and blocks * per >= n


@pytest.mark.parametrize("rows, columns, apart", [(1 << 20, 1 << 20, 0), (1 << 20, 1 << 20, 1),
                                                  (1 << 31, 500, 1), (1, 1 << 30, 0), (3, 5, 1),
                                                  ((1 << 32) - 1, 1, 1), (1000, 1001, 0)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_activations_of_any_size(driver, rows, columns, apart, dtype):  # noqa: F811
    for way in ("forward", "backward"):
        (rc, _, launches), = _launches(driver, f"gated_silu_{way},{rows},{columns},{dtype},{apart}")
        per = 8 if dtype == BF16 else 4
        least = rows * -(-columns // per) if apart or rows * columns > 1 << 30 else \
            -(-rows * columns // per)
        threads = sum(x * t for _, x, t in launches)
        assert rc == 0 and least <= threads < least + 256 * len(launches) + 1


@pytest.mark.parametrize("tensors, count", [(1, 1), (32, 50000), (33, 3), (96, 7), (97, 4096), (160, 5000), (161, 9),
                                            (338, 4500000), (65536, 4097), (2, 0)])
def test_launches_of_many_tensors(driver, tensors, count):  # noqa: F811
    """160 tensors a launch for the norm, 96 for the update, and a sum in the scratch for each
    block of the first."""
    some = tensors if count else -(-tensors // 3)
    for name, more in (("gradient_norm", 1), ("clip_gradients", -(-some // 96)),
                       ("sgd_step", -(-some // 96))):
        (rc, work, launches), = _launches(driver, f"{name},{tensors},{count},0,0")
        sums = [x for n, x, _ in launches if n.startswith("norm_sums")]
        assert rc == 0 and len(sums) == -(-some // 160) and work == 8 * sum(sums)
        assert len(launches) == len(sums) + more and max(x for _, x, _ in launches) <= 2048


def test_updates_in_place_and_shifted(driver):  # noqa: F811
    for name in ("clip_gradients", "sgd_step"):
        good, bad = _launches(driver, f"{name},5,100,1,0", f"{name},5,100,1,4")
        assert good[0] == 0 and good[2] and bad[0] == E_ARG and not bad[2]


def test_lists_that_find_no_memory_say_so(driver):  # noqa: F811
    """Each allocation of a call fails in turn: an error and its own text, not an earlier call's; and the
    scratch's size is answered all the same."""
    e_nomem = -1
    seen = {}
    for line in _run(driver.with_name("nomem")).splitlines():
        name, rc, work, text = line.split(" ", 3)
        seen.setdefault(name, []).append((int(rc), int(work), text.strip()))
    assert seen.keys() == {"gradient_norm", "clip_gradients", "sgd_step"}
    for name, calls in seen.items():
        assert calls[-1][0] == 0 and len(calls) > 1, name
        assert all(c[0] == e_nomem and c[2] == "out of memory" for c in calls[:-1]), (name, calls)
        assert {c[1] for c in calls} == {8 * 200}, name  # 200 chunks, a sum a block


@pytest.mark.parametrize("rows, columns, apart", [(1, (1 << 30) + 1, 0), (1, (1 << 32) - 1, 0), (2, (1 << 30) + 1, 0),
                                                  (3, (1 << 31) + 5, 1), (256, (1 << 32) - 1, 1)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_activations_of_rows_past_a_launch(driver, rows, columns, apart, dtype):  # noqa: F811
    """Rows of more than 2^30 values are taken in pieces: each value once."""
    for way in ("forward", "backward"):
        (rc, _, launches), = _launches(driver, f"gated_silu_{way},{rows},{columns},{dtype},{apart}")
        per = 8 if dtype == BF16 else 4
        threads = sum(x * t for _, x, t in launches)
        least = rows * -(-columns // per)
        assert rc == 0 and len(launches) == rows * -(-columns >> 30)
        assert least <= threads < least + 256 * len(launches)
