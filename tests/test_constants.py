"""Constants that calls share: they hold their values on every stream, inside and outside of captures."""

import pytest
import torch

import warpy_kernels as wk
from warpy_kernels_b200 import utils

FP8 = torch.float8_e4m3fn


def codes(*shape, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, device="cuda", generator=g).to(FP8)


def prefix_call(B, Hkv):
    q, kp, vp = codes(B, 2 * Hkv, 1, 64), codes(1, Hkv, 90, 64, seed=1), codes(1, Hkv, 90, 64, seed=2)
    k, v = codes(B, Hkv, 40, 64, seed=3), codes(B, Hkv, 40, 64, seed=4)
    names = ("q_descale", "k_descale", "v_descale", "k_prefix_descale", "v_prefix_descale")

    def run(ones=False):
        given = {n: torch.ones(1 if "prefix" in n else B, Hkv, device="cuda") for n in names} if ones else {}
        return wk.attn_fwd_shared_prefix(q, kp, vp, k, v, **given)

    return run


def forward_call(B, Hkv):
    q, k, v = codes(B, 2 * Hkv, 130, 64), codes(B, Hkv, 150, 64, seed=1), codes(B, Hkv, 150, 64, seed=2)
    return lambda ones=False: wk.attn_fwd(q, k, v, *([torch.ones(B, Hkv, device="cuda")] * 3 if ones else ()))


def backward_call(B, Hkv):
    q, k, v = codes(B, 2 * Hkv, 130, 64), codes(B, Hkv, 150, 64, seed=1), codes(B, Hkv, 150, 64, seed=2)
    ones_ = [torch.ones(B, Hkv, device="cuda")] * 3
    saved = wk.attn_fwd(q, k, v, *ones_)
    dout = torch.ones_like(saved[0])
    return lambda ones=False: wk.attn_bwd(q, k, v, *saved, dout, *(ones_ if ones else ()))


CALLS = [prefix_call, forward_call, backward_call]


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_first_use_of_descales_of_one_inside_a_capture(cuda, call):
    """A capture only records how they are filled: a call outside, before the graph runs, must not read them."""
    run = call(3, 11 + CALLS.index(call))  # a shape that no other call of the process has
    want = run(ones=True)
    junk = torch.full((1 << 22,), float("nan"), device="cuda")
    torch.cuda.synchronize()
    del junk
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    eager = run()
    assert all(torch.equal(x, y) for x, y in zip(eager, want))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(captured, want))
    # and once they are there, a capture uses them like any other call
    again = torch.cuda.CUDAGraph()
    with torch.cuda.graph(again):
        captured = run()
    again.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(captured, want))


@pytest.mark.gpu
@pytest.mark.parametrize("call", CALLS)
def test_first_use_of_descales_of_one_on_two_streams(cuda, call):
    """The second stream's call does not run before the first one's has filled them."""
    run = call(2, 17 + CALLS.index(call))
    want = run(ones=True)
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(one):
        torch.cuda._sleep(40_000_000)  # some 20 ms
        first = run()
    with torch.cuda.stream(two):
        second = run()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, want))
    assert all(torch.equal(x, y) for x, y in zip(second, want))


class _OnDevice:
    """Stands in for a tensor on a GPU and its stream."""

    is_cuda, device, waits = True, "cuda:0", 0

    def synchronize(self):
        self.waits += 1


def test_what_is_made_inside_a_capture_is_not_kept(monkeypatch):
    made = []

    def make():
        made.append(_OnDevice())
        return made[-1]

    class Device:
        def __init__(self, device):
            assert device == "cuda:0"

        def __enter__(self):
            pass

        def __exit__(self, *error):
            pass

    monkeypatch.setattr(utils, "_constants", {})
    monkeypatch.setattr(torch.cuda, "device", Device)
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: made[-1])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    first = utils.cached_tensor("key", make)
    assert utils.cached_tensor("key", make) is not first and all(x.waits == 0 for x in made)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    kept = utils.cached_tensor("key", make)
    assert kept.waits == 1 and utils.cached_tensor("key", make) is kept and kept.waits == 1
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert utils.cached_tensor("key", make) is kept
    host = utils.cached_tensor("other", lambda: torch.ones(2))  # on the host there is nothing to wait for
    assert utils.cached_tensor("other", lambda: None) is host


@pytest.mark.gpu
def test_graphs_that_run_beside_one_another_share_no_flags(cuda):
    """The forward marks query blocks to be computed again in a buffer that one call at a time may use."""
    from warpy_kernels_b200 import _lib

    host, graphs, seen = _lib.host(), [torch.cuda.CUDAGraph() for _ in range(2)], []
    g = torch.Generator(device="cuda").manual_seed(6)
    q, k, v = (torch.randn(2, 8, 700, 64, device="cuda", generator=g).bfloat16() for _ in range(3))
    k[:, :, 650] *= 60  # rows that rise beyond their reference's range
    want = wk.attn_fwd(q, k, v)
    outs = []
    for graph in graphs:  # on one stream, one after the other
        with torch.cuda.graph(graph):
            outs.append([wk.attn_fwd(q, k, v) for _ in range(2)])
            seen.append({host.block_flags(0, 64).data_ptr(), host.block_flags(0, 64).data_ptr()})
    seen.append({host.block_flags(0, 64).data_ptr()})
    assert all(len(x) == 1 for x in seen) and len(set.union(*seen)) == 3
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for stream, graph in zip(streams, graphs):
            with torch.cuda.stream(stream):
                graph.replay()
    assert all(torch.equal(x, y) for x, y in zip(wk.attn_fwd(q, k, v), want))
    torch.cuda.synchronize()
    for calls in outs:
        for got in calls:
            assert all(torch.equal(x, y) for x, y in zip(got, want))
