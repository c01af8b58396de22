"""Handles of the language-model operators: streams, threads, workspaces, status."""
import threading
import time

import numpy as np
import pytest
import torch

import infvino_b200 as ivb

pytestmark = pytest.mark.gpu
PER_THREAD = 2  # cudaStreamPerThread


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Call:
    """An attention call whose items are cut over CTAs, so that its joins use the workspace."""

    def __init__(self, seed, new, lens, heads=2, group=4, dim=64, page=32):
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-n // page) for n in lens]
        order, table, at = np.random.default_rng(seed).permutation(sum(need)), np.full((len(lens), max(need)), -1, np.int32), 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
        codes = [torch.randint(-127, 128, (at, heads, page, dim), generator=g, device="cuda").to(torch.int8) for _ in range(2)]
        scales = [2.0 ** torch.randint(-9, -4, (at, heads, page // 16), generator=g, device="cuda").float() for _ in range(2)]
        self.cache, self.table, self.max_new = ivb.KvCache(*codes, *scales), ints(table), max(new)
        self.q = torch.randn((sum(new), heads * group, dim), generator=g, device="cuda").half()
        self.out = torch.empty_like(self.q)
        self.offsets, self.lens = ints([0] + list(np.cumsum(new))), ints(lens)

    def run(self, ops, st, out=None):
        ops.attend(self.cache, self.q, self.out if out is None else out, self.offsets, self.lens, self.table, max_new=self.max_new, stream=st)

    def expected(self):
        want = torch.empty_like(self.q)
        with ivb.KvOps(0) as ops:
            self.run(ops, stream(), want)
            ops.synchronize(stream())
        return want


def test_per_thread_streams_have_their_own_workspaces():
    """cudaStreamPerThread is one handle value, but another stream in every thread."""
    calls = [Call(1, [1, 1], [9000, 5000]), Call(2, [1, 1, 1], [4000, 7000, 100]), Call(3, [300], [3000]), Call(4, [200, 100], [900, 2000])]
    wants = [c.expected() for c in calls]
    torch.cuda.synchronize()
    wrong = []
    with ivb.KvOps(0) as ops:
        def work(c, want):
            outs = [torch.empty_like(c.q) for _ in range(40)]
            torch.cuda.synchronize()
            for o in outs:
                c.run(ops, PER_THREAD, o)
            ops.synchronize(PER_THREAD)
            wrong.append(sum(not torch.equal(o, want) for o in outs))

        threads = [threading.Thread(target=work, args=z) for z in zip(calls, wants)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert wrong == [0] * len(calls)


def test_a_capture_without_a_call_before_is_refused():
    c = Call(5, [1, 1], [500, 300])
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    with ivb.KvOps(0) as ops:
        ops.reserve(other.cuda_stream)
        torch.cuda.synchronize()
        graph, refused = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(graph, stream=side):
            try:
                c.run(ops, side.cuda_stream)
            except ivb.NativeError as e:
                refused.append((e.status, e.message))
            c.out.zero_()  # (a graph of something)
        assert len(refused) == 1 and refused[0][0] == 1 and "ivc_kv_reserve" in refused[0][1]
        ops.reserve(side.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            c.run(ops, side.cuda_stream)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.out, c.expected())


def test_release_gives_the_workspace_back():
    c = Call(6, [1, 1, 30], [700, 3000, 400])
    want = c.expected()
    streams = [torch.cuda.Stream() for _ in range(6)]
    with ivb.KvOps(0) as ops:
        for s in streams[:1]:  # (what the first call of all brings with it)
            c.run(ops, s.cuda_stream)
            ops.release(s.cuda_stream)
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        for _ in range(2):
            for s in streams:
                ops.reserve(s.cuda_stream)
            held = before - torch.cuda.mem_get_info()[0]
            assert held > 6 << 20
            for s in streams:
                c.out.zero_()
                torch.cuda.synchronize()
                c.run(ops, s.cuda_stream)
                ops.release(s.cuda_stream)  # (waits)
                assert torch.equal(c.out, want)
                ops.release(s.cuda_stream)  # nothing is left to free
            assert torch.cuda.mem_get_info()[0] >= before - held // 6
        c.run(ops, streams[0].cuda_stream)
        ops.synchronize(streams[0].cuda_stream)
        assert torch.equal(c.out, want)


@pytest.mark.parametrize("dim", [64, 128])
def test_calls_after_a_timed_out_one(dim):
    """Every other CTA of a prompt call gives up: it is reported, and later calls on the same workspace give the bits they would have given."""
    many = [Call(7, [300], [3000], dim=dim), Call(8, [40, 500, 1], [900, 2000, 3], dim=dim), Call(9, [700], [700], heads=3, group=1, dim=dim),
            Call(11, [1000], [1500], heads=8, group=8, dim=dim)]  # (the last: shares that end one cut item and begin another)
    few = Call(10, [1, 1], [9000, 300], dim=dim)
    wants = [c.expected() for c in many + [few]]
    L, st = ivb._native.lib(), stream()
    with ivb.KvOps(0) as ops:
        for c in many:
            assert L.ivc_debug_kv_probe(ops._h, 2_000_000) == 0
            for _ in range(3):  # (odd: of two parts one is missing each time)
                c.run(ops, st)
                with pytest.raises(ivb.NativeError) as e:
                    ops.synchronize(st)
                assert e.value.status == 5 and "timed out" in e.value.message
            assert L.ivc_debug_kv_probe(ops._h, 0) == 0
            for d, want in zip(many + [few], wants):
                for _ in range(2):
                    d.out.fill_(float("nan"))
                    d.run(ops, st)
                    ops.synchronize(st)
                    assert torch.equal(d.out, want)
        assert L.ivc_debug_kv_probe(ops._h, -1) == 1


def test_waiting_for_one_stream_does_not_hold_up_calls_on_another():
    c = Call(12, [1, 1], [500, 300])
    want = c.expected()
    slow, fast = torch.cuda.Stream(), torch.cuda.Stream()
    with ivb.KvOps(0) as ops:
        c.run(ops, fast.cuda_stream)  # (its workspace)
        c.out.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(slow):
            torch.cuda._sleep(2_000_000_000)  # about a second
        entered, done = threading.Event(), threading.Event()

        def wait():
            entered.set()
            ops.synchronize(slow.cuda_stream)
            done.set()

        t = threading.Thread(target=wait)
        t.start()
        entered.wait()
        time.sleep(0.1)
        c.run(ops, fast.cuda_stream)
        fast.synchronize()
        first = not done.is_set()
        t.join()
        assert first, "the call waited for the other stream"
        assert torch.equal(c.out, want)


def test_threads_share_a_handle():
    """Calls, errors and waits from several threads at once, each on a stream of its own."""
    calls = [Call(20 + i, [1, 1, 40], [3000, 500, 900]) for i in range(4)]
    wants = [c.expected() for c in calls]
    wrong = []
    with ivb.KvOps(0) as ops:
        def work(c, want):
            try:
                calls_of(c, want)
            except Exception as e:
                wrong.append(repr(e))

        def calls_of(c, want):
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for _ in range(30):
                    c.out.zero_()
                    c.run(ops, s.cuda_stream)
                    try:
                        ops.attend(c.cache, c.q, c.out, c.offsets, c.lens, c.table, max_new=0, stream=s.cuda_stream)
                        wrong.append("not refused")
                    except ivb.NativeError as e:
                        if e.status != 1 or "max_new" not in e.message:
                            wrong.append(str(e))
                    ops.synchronize(s.cuda_stream)
                    if not torch.equal(c.out, want):
                        wrong.append("other bits")

        threads = [threading.Thread(target=work, args=z) for z in zip(calls, wants)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not wrong, wrong[:3]


def test_a_new_handle_keeps_errors_while_the_default_stream_is_busy():
    table = torch.zeros((4, 32, 2), device="cuda")
    x, pos = torch.zeros((1, 1, 64), dtype=torch.float16, device="cuda"), ints([9])
    side = torch.cuda.Stream()
    with ivb.KvOps(0) as ops:  # (what the first calls of all bring with them)
        ops.rope(x, x, ivb.Rotary(table), ints([1]), stream=side.cuda_stream)
        ops.synchronize(side.cuda_stream)
    torch.cuda.synchronize()
    torch.cuda._sleep(600_000_000)  # some 0.3 s of the default stream
    with ivb.KvOps(0) as ops:
        ops.rope(x, x, ivb.Rotary(table), pos, stream=side.cuda_stream)
        side.synchronize()
        torch.cuda.synchronize()
        with pytest.raises(ivb.NativeError) as e:
            ops.synchronize(side.cuda_stream)
        assert e.value.status == 5 and "rotary table" in e.value.message


@pytest.mark.parametrize("other", [0, 1])  # the legacy stream's two names
def test_the_default_stream_while_another_is_captured(other):
    """A call on the default stream beside a capture runs; release of the captured stream is refused and does no harm."""
    c, d = Call(30, [1, 1], [900, 300]), Call(31, [50], [400])
    wants = [c.expected(), d.expected()]
    side = torch.cuda.Stream()
    with ivb.KvOps(0) as ops:
        c.run(ops, 0)
        ops.reserve(side.cuda_stream)
        torch.cuda.synchronize()
        c.out.zero_()
        torch.cuda.synchronize()
        graph, errors = torch.cuda.CUDAGraph(), []
        with torch.cuda.graph(graph, stream=side):
            d.run(ops, side.cuda_stream)
            for what in (lambda: c.run(ops, other), lambda: ops.release(side.cuda_stream)):
                try:
                    what()
                    errors.append(None)
                except ivb.NativeError as e:
                    errors.append(e.status)
        graph.replay()
        torch.cuda.synchronize()
        assert errors == [None, 1]
        assert torch.equal(c.out, wants[0]) and torch.equal(d.out, wants[1])


def test_closed_handles_and_lone_queries_are_refused():
    c = Call(40, [1], [40])
    k = torch.zeros((1, 2, 64), dtype=torch.float16, device="cuda")
    rotary, pos = ivb.Rotary(torch.zeros((50, 32, 2), device="cuda")), ints([39])
    ops = ivb.KvOps(0)
    for lone in (dict(q=c.q), dict(q_out=c.out)):
        with pytest.raises(ValueError, match="q_out"):
            ops.append(c.cache, k, k, c.offsets, ints([39]), c.table, rotary=rotary, pos=pos, stream=stream(), **lone)
    ops.close()
    for call in (lambda: c.run(ops, stream()), lambda: ops.synchronize(stream()), lambda: ops.rope(k, k, rotary, pos, stream()), lambda: ops.release(stream())):
        with pytest.raises(ValueError, match="closed"):
            call()
