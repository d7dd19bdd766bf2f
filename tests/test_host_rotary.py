"""`matricxon_amd.rotary` and `mxa_rope` without a GPU: the frequency tables and what is refused."""

import ctypes
import math

import pytest
import torch

from matricxon_amd.rotary import HipRotary, rotary_frequencies


def test_plain_and_linear_tables() -> None:
    f, m = rotary_frequencies(8, 10000.0)
    assert m == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    g, _ = rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(g, f / 4)
    h, _ = rotary_frequencies(8, 10000.0, None, torch.tensor([1.0, 2.0, 4.0, 8.0]))
    assert torch.equal(h, f / torch.tensor([1, 2, 4, 8], dtype=torch.float64))


def test_ntk_stretches_the_last_pair_by_the_factor() -> None:
    """base' = base factor^(d / (d - 2)): the first pair keeps its frequency, the last one is divided by the factor."""
    d, factor = 64, 8.0
    f, _ = rotary_frequencies(d)
    g, _ = rotary_frequencies(d, scaling={"type": "ntk", "factor": factor})
    assert g[0] == f[0] and math.isclose(g[-1] * factor, f[-1], rel_tol=1e-12)


@pytest.mark.parametrize("scaling", [
    {"type": "yarn", "factor": 16.0, "original_context": 4096},
    {"type": "llama3", "factor": 16.0, "original_context": 4096},
    {"type": "llama3", "factor": 4.0, "original_context": 8192, "low_freq_factor": 2.0, "high_freq_factor": 8.0},
], ids=lambda s: s["type"])
def test_bands(scaling) -> None:
    """Fast pairs keep their frequency, slow ones are divided by the factor, none lies outside, in order."""
    d, factor, context = 128, scaling["factor"], scaling["original_context"]
    f, _ = rotary_frequencies(d)
    g, m = rotary_frequencies(d, scaling=scaling)
    turns = f * context / (2 * math.pi)
    fast, slow = (33, 0.99) if scaling["type"] == "yarn" else (scaling.get("high_freq_factor", 4.0),
                                                              scaling.get("low_freq_factor", 1.0))
    assert torch.equal(g[turns >= fast], f[turns >= fast])
    # yarn's ramp ends at the next whole pair behind the last that turns once
    assert torch.allclose(g[turns <= 0.8 * slow], f[turns <= 0.8 * slow] / factor, rtol=1e-13, atol=0)
    assert (g <= f).all() and (g >= f / factor * (1 - 1e-13)).all() and (g[1:] < g[:-1]).all()
    assert math.isclose(m, 0.1 * math.log(factor) + 1 if scaling["type"] == "yarn" else 1.0)


def test_bad_tables_are_refused() -> None:
    for args, match in (((7,), "even"), ((0,), "even"), ((8, -1.0), "base"), ((8, 1e4, {"type": "x"}), "type"),
                        ((8, 1e4, {"factor": 2.0}), "type"), ((8, 1e4, {"type": "linear"}), "needs"),
                        ((8, 1e4, {"type": "yarn", "factor": 2.0}), "original_context"),
                        ((8, 1e4, {"type": "linear", "factor": 2.0, "beta_fast": 1}), "beta_fast"),
                        ((8, 1e4, {"type": "linear", "factor": 0.0}), "positive"),
                        ((2, 1e4, {"type": "ntk", "factor": 2.0}), "ntk"),
                        ((8, 1e4, {"type": "llama3", "factor": 2.0, "original_context": 9, "low_freq_factor": 5.0}), "low"),
                        ((8, 1.0, {"type": "yarn", "factor": 2.0, "original_context": 9}), "base"),
                        ((8, 1e4, None, torch.ones(3)), "freq_factors")):
        with pytest.raises(ValueError, match=match):
            rotary_frequencies(*args)
    for args in ((7, {}), (64, {"rotary_dim": 66}), (64, {"rotary_dim": 0}), (64, {"rotary_dim": 7}), (2048, {})):
        with pytest.raises(ValueError):
            HipRotary(args[0], device="cpu", **args[1])
    with pytest.raises(ValueError, match="HIP device"):
        HipRotary(64, device="cpu")(torch.zeros(1, 2, 64), None, torch.zeros(1, dtype=torch.int64))


def test_argument_errors_return_status_without_launching() -> None:
    from matricxon_amd import _lib

    lib = _lib.load()
    vp = ctypes.c_void_p
    a, st = vp(0x10000), (ctypes.c_longlong * 3)(0, 1024, 64)

    def call(q=a, qs=st, hq=4, k=a, ks=st, hk=2, pos=a, pos64=1, turns=a, n=3, seq=3, dim=64, rot=64, bf16=1, q_out=a,
             k_out=a):
        return lib.mxa_rope(q, qs, hq, k, ks, hk, pos, pos64, 0, 1, turns, n, seq, dim, rot, 0, 1.0, bf16, q_out, k_out,
                            None)

    for bad in (dict(q=None), dict(qs=None), dict(hq=0), dict(hq=65537), dict(hk=-1), dict(hk=65537), dict(k=None),
                dict(ks=None), dict(k_out=None), dict(q_out=None), dict(pos=None), dict(turns=None), dict(n=0),
                dict(seq=0), dict(dim=0), dict(dim=63, rot=62), dict(dim=1026, rot=64), dict(rot=0), dict(rot=66),
                dict(rot=63), dict(q=vp(0x10001)), dict(bf16=0, q=vp(0x10002)), dict(k=vp(0x10001)),
                dict(q_out=vp(0x10001)), dict(k_out=vp(0x10001)), dict(pos=vp(0x10004)), dict(pos64=0, pos=vp(0x10002)),
                dict(turns=vp(0x10004))):
        assert call(**bad) == -1, bad


def test_more_tokens_than_a_grid_holds_are_refused() -> None:
    from matricxon_amd import _lib

    a, st = ctypes.c_void_p(0x10000), (ctypes.c_longlong * 3)(0, 2, 2)
    for n in ((1 << 24) + 1, 2 ** 31 - 1):
        assert _lib.load().mxa_rope(a, st, 1, None, None, 0, a, 1, 0, 1, a, n, n, 2, 2, 0, 1.0, 1, a, None, None) == -1


def test_the_table_is_made_on_the_host_under_any_default_device() -> None:
    want, _ = rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 8.0, "original_context": 4096})
    with torch.device("meta"):  # as torch.set_default_device sets one
        f, _ = rotary_frequencies(64, 1e4, {"type": "yarn", "factor": 8.0, "original_context": 4096})
        g, _ = rotary_frequencies(8, 1e4, None, torch.ones(4, device="cpu"))
    assert f.device.type == g.device.type == "cpu" and torch.equal(f, want)
