"""`mxa_moe_layer`, `mxa_moe_topk` and `mxa_moe_combine_masked` without a GPU: what they take and what they refuse, with
nothing launched."""

import ctypes

Q8_0, Q4_K, Q6_K, IQ4_XS = 8, 12, 14, 23


def load():
    from matricxon_amd import _lib

    return _lib.load()


def test_what_the_layer_takes() -> None:
    size = load().mxa_moe_layer_workspace_bytes
    for args in ((Q4_K, Q6_K, 8, 2, 1, 4096, 14336, 1), (Q8_0, Q8_0, 256, 8, 8, 256, 256, 0),
                 (Q6_K, Q4_K, 16, 16, 4, 16384, 16384, 1)):
        assert size(*args) > 0, args
    good = (Q4_K, Q6_K, 8, 2, 4, 4096, 1024, 1)
    for at, value in ((0, IQ4_XS), (0, 10), (1, IQ4_XS), (2, 0), (2, 257), (2, 1), (3, 0), (3, 9), (4, 0), (4, 9),
                      (5, 300), (5, 0), (5, 65 * 256), (6, 300), (6, 0), (6, 65 * 256)):
        args = list(good)
        args[at] = value
        assert size(*args) == 0, args
    assert size(Q4_K, Q6_K, 40, 9, 8, 4096, 1024, 1) == 0  # 72 pairs


def test_argument_errors_return_status_without_launching() -> None:
    lib = load()
    vp = ctypes.c_void_p
    a = vp(0x10000)  # a well-aligned stand-in: nothing is dereferenced on these paths
    gate_stride, down_stride = 512 * 144, 256 * 420

    def layer(gt=Q4_K, dt=Q6_K, gate=a, up=a, gs=gate_stride, down=a, ds=down_stride, e=4, x=a, logits=a, lb=0, k=2, t=1,
              embd=256, ffn=512, ids=a, w=a, out=a, ob=1, ws=a, ws_bytes=1 << 20):
        return lib.mxa_moe_layer(gt, dt, gate, up, gs, down, ds, e, x, 1, logits, lb, k, 1, 1.0, t, embd, ffn, 0, ids, w, out,
                                 ob, ws, ws_bytes, None)

    for bad in (dict(gt=IQ4_XS), dict(gate=None), dict(up=None), dict(down=None), dict(x=None), dict(logits=None),
                dict(ids=None), dict(w=None), dict(out=None), dict(k=5), dict(t=9), dict(t=0), dict(embd=300),
                dict(gate=vp(0x10008)), dict(up=vp(0x10004)), dict(down=vp(0x10002)), dict(x=vp(0x10008)),
                dict(logits=vp(0x10002)), dict(lb=1, logits=vp(0x10001)), dict(ids=vp(0x10002)), dict(w=vp(0x10002)),
                dict(out=vp(0x10001)), dict(ob=0, out=vp(0x10002)), dict(gs=gate_stride - 16), dict(ds=down_stride - 16),
                dict(gs=gate_stride + 4), dict(ds=down_stride + 8), dict(ws=vp(0x10008))):
        assert layer(**bad) == -1, bad
    assert layer(ws=None) == -2 and layer(ws_bytes=100) == -2

    def topk(logits=a, lb=0, t=2, e=8, k=2, ids=a, w=a):
        return lib.mxa_moe_topk(logits, lb, t, e, k, 1, 1.0, ids, w, None)

    for bad in (dict(logits=None), dict(ids=None), dict(w=None), dict(logits=vp(0x10002)), dict(lb=1, logits=vp(0x10001)),
                dict(t=0), dict(e=0), dict(e=257), dict(k=0), dict(k=9), dict(e=100, k=65)):
        assert topk(**bad) == -1, bad

    def combine(down=a, ids=a, w=a, t=2, k=2, n=256, out=a):
        return lib.mxa_moe_combine_masked(down, None, ids, w, t, k, n, 1, out, None)

    for bad in (dict(down=None), dict(ids=None), dict(w=None), dict(out=None), dict(t=0), dict(k=17), dict(n=0)):
        assert combine(**bad) == -1, bad


def test_more_tokens_than_a_grid_holds_are_refused() -> None:
    a = ctypes.c_void_p(0x10000)
    for t in ((1 << 24) + 1, 2 ** 31 - 1):
        assert load().mxa_moe_topk(a, 0, t, 8, 2, 1, 1.0, a, a, None) == -1


def test_masked_routing_refuses_bad_arguments_without_launching() -> None:
    lib, a = load(), ctypes.c_void_p(0x10000)

    def call(ids=a, t=2, k=2, e=8, offsets=a, pair_tok=a, rows=a):
        return lib.mxa_moe_route_masked(ids, 0, t, k, e, offsets, pair_tok, rows, None, None)

    for bad in (dict(ids=None), dict(offsets=None), dict(pair_tok=None), dict(rows=None), dict(t=0), dict(k=0),
                dict(e=0), dict(e=257), dict(t=1 << 18, k=5)):
        assert call(**bad) == -1, bad


def test_experts_moved_to_the_host_are_refused() -> None:
    """What `module.cpu()` leaves: a layer whose host addresses may not reach a kernel."""
    import pytest
    import torch

    from matricxon_amd.moe import HipPackedMoEExperts

    mod = HipPackedMoEExperts.__new__(HipPackedMoEExperts)
    torch.nn.Module.__init__(mod)
    for name in ("gate_packed", "up_packed", "down_packed"):
        mod.register_buffer(name, torch.zeros(4, 256, 144, dtype=torch.uint8))
    mod.n_embd, mod.num_experts, mod.dtype, mod._gemm = 256, 4, torch.float32, None
    with pytest.raises(ValueError, match="HIP device"):
        mod.forward_logits(torch.zeros(2, 256), torch.zeros(2, 4), 2)


def test_experts_of_other_shapes_do_not_reach_the_layer_call() -> None:
    """up of fewer rows than gate, down of fewer experts' bytes, other dtypes: not what `mxa_moe_layer` assumes."""
    import torch
    import torch.nn.functional as F

    from matricxon_amd.moe import HipPackedMoEExperts

    def layer(gate=(4, 512, 144), up=(4, 512, 144), down=(4, 256, 288), dtype=torch.uint8):
        w = [torch.zeros(s, dtype=dtype) for s in (gate, up, down)]
        return HipPackedMoEExperts(*w, Q4_K, Q4_K, Q4_K, 256, 512, F.silu)

    assert layer()._layer_ok
    for bad in (dict(gate=(4, 256, 144)), dict(up=(4, 256, 144)), dict(up=(4, 512, 160)), dict(down=(4, 128, 288)),
                dict(down=(4, 256, 144)), dict(dtype=torch.int8)):
        assert not layer(**bad)._layer_ok, bad


def test_every_launch_goes_to_the_device_of_the_experts(monkeypatch) -> None:
    """Experts on a device that is not the current one: the grouped launches, too, run with theirs as the current one."""
    import contextlib

    import pytest
    import torch

    from matricxon_amd import moe

    current, seen = [0], []

    @contextlib.contextmanager
    def device(d):
        kept, current[0] = current[0], d.index
        try:
            yield
        finally:
            current[0] = kept

    class OnDevice1(torch.Tensor):  # host values that say they are on the second device
        device, is_cuda = torch.device("cuda", 1), True

    def there(*shape):
        return torch.zeros(*shape).as_subclass(OnDevice1)

    class Gemm:
        @staticmethod
        def _check_router(*_):
            pass

        @staticmethod
        def moe_topk(logits, top_k, *_):
            seen.append(current[0])
            return there(len(logits), top_k), there(len(logits), top_k)

    monkeypatch.setattr(moe, "_elsewhere", lambda d: d.index != current[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    mod = moe.HipPackedMoEExperts.__new__(moe.HipPackedMoEExperts)
    torch.nn.Module.__init__(mod)
    mod._buffers["gate_packed"] = there(4, 256, 144)
    mod.n_embd, mod.num_experts, mod.dtype, mod._gemm = 256, 4, torch.float32, Gemm
    mod._few_tokens = lambda *_: seen.append(current[0])
    mod._grouped = lambda x, *_, **__: (seen.append(current[0]), x)[1]
    for tokens in (3, 20):
        out, _, _ = mod.forward_logits(there(tokens, 256), there(tokens, 4), 2)
        assert out.shape == (tokens, 256) and seen == [1, 1, 1] and current == [0], seen
        seen.clear()
    with pytest.raises(ValueError, match="reciprocal"):
        mod.forward_logits(there(20, 256), there(20, 4), 2, q8k_scale="reciprocal")
    assert set(seen) == {1} and current == [0]
