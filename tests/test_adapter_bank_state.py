"""What an AdapterBank keeps between calls -- the bf16 stacks that the kernels read -- under streams, threads, captures and optimizers: a call sees the
parameters as they are, whoever laid the stacks out.  Comparisons are bit for bit with a bank that was made from the same weights."""
import threading
import time

import pytest
import torch

from aqualora_amd import adapters, inference, ksamplers, ops
from aqualora_amd.unet import lora_keys
from tests.common import ppft_inputs, tiny_lora, tiny_unet

DEV = "cuda"
SLEEP = 50_000_000     # cycles: 20 ms or more, longer than the host needs for what is queued behind it
gpu = pytest.mark.gpu


class Site:
    """A small projection with three adapters, and banks of two sets of weights."""

    def __init__(self, seed=0):
        gen = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(s, generator=gen)  # noqa: E731
        K, N, r, G = 320, 256, 16, 3
        bf = torch.bfloat16
        self.packed = ops.PackedLinear(rn(N, K).to(DEV) / K ** 0.5, rn(N).to(DEV))
        self.old, self.new = ((rn(G, r, K).to(bf).float() / r, (0.2 * rn(G, N, r)).to(bf).float()) for _ in range(2))
        self.plan = adapters.RequestPlan([0, 2, -1, 1], [70, 1, 30, 99])
        self.x, self.dy = rn(200, K).to(DEV, bf), rn(200, N).to(DEV, bf)

    def bank(self, weights, trainable=True):
        return adapters.AdapterBank(*weights, ranks=[16, 12, 16], scales=[1.0, 0.5, 1.25], trainable=trainable)

    def call(self, bank):
        return ops.adapter_linear(self.x, self.packed, bank, self.plan)

    def step(self, bank):
        x = self.x.detach().requires_grad_(True)
        y = ops.adapter_linear(x, self.packed, bank, self.plan)
        return (y.detach(),) + torch.autograd.grad(y, (x, bank.down, bank.up), self.dy)


def put(bank, weights):
    """An eager step of an optimizer."""
    with torch.no_grad():
        bank.down.copy_(weights[0])
        bank.up.copy_(weights[1])


def same(a, b):
    return all(torch.equal(x, y) for x, y in zip(a, b))


@gpu
def test_other_streams_wait_for_a_layout():
    """The parameters change, both streams are ordered behind that; one stream's call lays the bank out (late: its stream is busy), the other's call comes next."""
    s = Site()
    bank = s.bank(s.old)
    want = s.step(s.bank(s.new))
    new = [w.to(DEV) for w in s.new]
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for first, second in ((one, two), (torch.cuda.current_stream(), one), (two, torch.cuda.current_stream())):
        put(bank, [w.to(DEV) for w in s.old])
        s.step(bank)
        put(bank, new)
        torch.cuda.synchronize()
        with torch.cuda.stream(first):
            torch.cuda._sleep(SLEEP)
            a = s.step(bank)
        with torch.cuda.stream(second):
            b = s.step(bank)
        torch.cuda.synchronize()
        assert same(a, want) and same(b, want)


@gpu
def test_a_layout_waits_for_the_streams_that_still_read():
    """A stream is late with its pass over the old weights; another stream's call lays the new ones out."""
    s = Site(1)
    old, new = s.step(s.bank(s.old)), s.step(s.bank(s.new))
    to = [w.to(DEV) for w in s.new]
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    for late, next_ in ((one, two), (torch.cuda.current_stream(), one), (one, torch.cuda.current_stream())):
        bank = s.bank(s.old)
        s.call(bank)
        torch.cuda.synchronize()
        with torch.cuda.stream(late):
            torch.cuda._sleep(SLEEP)
            a = s.step(bank)
        with torch.cuda.stream(next_):
            put(bank, to)
            b = s.step(bank)
        torch.cuda.synchronize()
        assert same(a, old) and same(b, new)


@gpu
def test_threads_come_together_after_a_step():
    """Two threads, each with a stream of its own, call forward and backward right after the parameters changed: one layout, no pass refused, the new weights in both."""
    s = Site(2)
    bank = s.bank(s.old)
    weights = [[w.to(DEV) for w in ws] for ws in (s.old, s.new)]
    want = [s.step(s.bank(ws)) for ws in (s.old, s.new)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    barrier, got, errors = threading.Barrier(3), [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(streams[i]):
                for _ in range(60):
                    barrier.wait(60)
                    got[i] = s.step(bank)
                    torch.cuda.current_stream().synchronize()
                    barrier.wait(60)
        except Exception as e:  # noqa: BLE001
            errors.append(e)
            barrier.abort()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    try:
        for k in range(60):
            put(bank, weights[(k + 1) % 2])
            serial = bank.handle.serial
            torch.cuda.synchronize()
            barrier.wait(60)
            barrier.wait(60)
            assert bank.handle.serial == serial + 1
            assert all(same(g, want[(k + 1) % 2]) for g in got), k
    except threading.BrokenBarrierError:
        pass
    except AssertionError:
        barrier.abort()
        raise
    finally:
        for t in threads:
            t.join()
    assert not errors, errors


@gpu
def test_a_change_under_a_layout_is_not_lost():
    """The versions that a layout has seen are those from before its copies: a parameter changed right behind them is laid out by the next call."""
    s = Site(3)
    bank = s.bank(s.old)
    new = [w.to(DEV) for w in s.new]

    class Late:                                          # the handle, with another thread's write between the copies and their end
        def __getattr__(self, name):
            return getattr(handle, name)

        def end_layout(self):
            put(bank, new)
            handle.end_layout()
    handle = bank.handle
    bank.handle = Late()
    bank.refresh(force=True)
    bank.handle = handle
    assert torch.equal(s.call(bank), s.call(s.bank(s.new)))


@gpu
def test_a_layout_from_inside_a_call_is_refused():
    s = Site(4)
    bank = s.bank(s.old)

    def pack(t):
        bank.refresh(force=True)
        return t
    x = s.x.detach().requires_grad_(True)
    with pytest.raises(RuntimeError, match="inside a call"):
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            ops.adapter_linear(x, s.packed, bank, s.plan)
    assert torch.equal(s.call(bank), s.call(s.bank(s.old)))


@gpu
def test_transposed_stacks_are_there_when_they_are_complete():
    """One thread's call lays a frozen bank's transposed stacks out on a busy stream; another thread's call comes meanwhile."""
    s = Site(5)

    def step(bank):
        x = s.x.detach().requires_grad_(True)
        return torch.autograd.grad(ops.adapter_linear(x, s.packed, bank, s.plan), x, s.dy)
    want = step(s.bank(s.old, False))
    bank = s.bank(s.old, False)
    torch.cuda.synchronize()
    got = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(5):
                torch.cuda._sleep(SLEEP)
            got.append(step(bank))
            torch.cuda.current_stream().synchronize()
    thread = threading.Thread(target=work)
    thread.start()
    time.sleep(0.02)
    with torch.cuda.stream(torch.cuda.Stream()):
        got.append(step(bank))
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 2 and all(same(g, want) for g in got)


@gpu
def test_a_capture_that_finds_the_bank_stale_is_refused():
    s = Site(6)
    bank = s.bank(s.old)
    want = s.call(s.bank(s.new))
    s.call(bank)
    put(bank, [w.to(DEV) for w in s.new])
    torch.cuda.synchronize()
    with torch.no_grad():
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                s.call(bank)
        torch.cuda.synchronize()
        assert torch.equal(s.call(bank), want)           # nothing was marked
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):                    # and now there is nothing to lay out
            bank.refresh()
            y = s.call(bank)
    for weights in (s.old, s.new, s.old):                # eager steps between the replays
        put(bank, [w.to(DEV) for w in weights])
        bank.refresh()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, s.call(s.bank(weights)))


@gpu
@pytest.mark.parametrize("aborted", [False, True])
def test_a_layout_in_a_capture_is_for_its_replays(aborted):
    s = Site(7)
    bank = s.bank(s.old)
    old, new = (s.call(s.bank(w)) for w in (s.old, s.new))
    s.call(bank)
    to = [w.to(DEV) for w in s.new]
    put(bank, to)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad():
        try:
            with torch.cuda.graph(graph):
                bank.refresh(force=True)
                y = s.call(bank)
                if aborted:
                    raise KeyError
        except KeyError:
            pass
        torch.cuda.synchronize()
        assert torch.equal(s.call(bank), new)            # eager, ahead of the first replay
        if aborted:
            return
        for weights, want in ((s.old, old), (s.new, new)):
            for p, w in zip((bank.down, bank.up), weights):
                p.data.copy_(w.to(DEV))                  # (no version tells of it)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(y, want) and torch.equal(s.call(bank), want)


@gpu
def test_two_training_steps_in_one_graph():
    s = Site(8)
    lr = 0.05

    def two(bank):
        out = []
        for _ in range(2):
            y = s.call(bank)
            out += [y.detach(), *torch.autograd.grad(y, (bank.down, bank.up), s.dy)]
            with torch.no_grad():
                bank.down.sub_(lr * out[-2])
                bank.up.sub_(lr * out[-1])
            bank.refresh(force=True)
        return out
    eager, bank = s.bank(s.old), s.bank(s.old)
    two(eager), two(bank)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = two(bank)
    for k in range(3):
        want = two(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert same(got, want), k
        assert torch.equal(s.call(bank), s.call(eager))


@gpu
@pytest.mark.parametrize("kind", ["single", "foreach", "fused"])
@pytest.mark.parametrize("name", ["SGD", "Adam", "AdamW"])
def test_a_bank_follows_every_form_of_an_optimizer(name, kind):
    s = Site(9)
    bank = s.bank(s.old)
    opt = getattr(torch.optim, name)(bank.parameters(), lr=0.05, foreach=kind == "foreach", fused=kind == "fused")
    for _ in range(3):
        y = s.call(bank)
        assert torch.equal(y, s.call(s.bank((bank.down.detach(), bank.up.detach()))))
        before = bank.up.detach().clone()
        bank.down.grad, bank.up.grad = torch.autograd.grad(y, (bank.down, bank.up), s.dy)
        opt.step()
        assert not torch.equal(bank.up.detach(), before)


def test_fused_steps_raise_the_versions_of_bank_weights_only():
    ps = [torch.nn.Parameter(torch.ones(4)) for _ in range(3)]
    for p in ps[:2]:
        p.grad = torch.ones(4)
    ps[0]._aql_bank_weights = ps[2]._aql_bank_weights = True
    opt = torch.optim.SGD(ps, lr=0.1, fused=True)
    opt.register_step_post_hook(adapters._count_fused_step)
    opt.step()
    assert [p._version for p in ps] == [1, 0, 0] and all((p < 1).all() for p in ps[:2])      # (no gradient, no step)


@gpu
def test_a_sampling_machine_follows_the_banks():
    """A second run of one machine: after a step on the banks, and after other banks were attached."""
    unet = tiny_unet(DEV, torch.bfloat16)
    keys = lora_keys(unet)
    loras = [{f"{k}.{n}.weight": t for k, p in tiny_lora(keys, unet, rank=8, up_std=std).items() for n, t in zip(("down", "up"), p)} for std in (0.1, 0.2)]
    inp = ppft_inputs(B=2, device=DEV)
    unc = torch.zeros_like(inp["ctx"])
    prog = ksamplers.program("euler", 3)
    new = lambda: ksamplers.SamplerMachine(unet, inp["ctx"], unc, inp["z"], 3.0, scale=adapters.RequestPlan([1, 0]))  # noqa: E731

    def again(m):
        m.x.copy_(inp["z"])
        return m.run(prog)
    banks = inference.attach_adapters(unet, loras, trainable=True)
    m = new()
    first = m.run(prog)
    assert torch.equal(again(m), first)
    with torch.no_grad():
        for bank in banks.values():
            bank.up.mul_(0.5)
    second = again(m)
    assert torch.equal(second, new().run(prog)) and not torch.equal(second, first)
    inference.attach_adapters(unet, loras[::-1])
    third = again(m)
    assert torch.equal(third, new().run(prog)) and not torch.equal(third, first)


@gpu
@pytest.mark.parametrize("trainable", [False, True])
def test_bank_and_plan_dropped_while_a_stream_still_reads(trainable):
    """Made on one stream, used late on another and dropped at once: their memory is not given out again before that."""
    s = Site(10)
    x = s.x.detach().requires_grad_(True)
    want = [ops.adapter_linear(x, s.packed, s.bank(s.new), s.plan)]
    want = [want[0].detach(), *torch.autograd.grad(want[0], x, s.dy)]
    torch.cuda.synchronize()
    for _ in range(3):
        bank, plan = s.bank(s.new, trainable), adapters.RequestPlan([0, 2, -1, 1], [70, 1, 30, 99])
        sizes = [t.numel() * t.element_size() for t in (bank.handle.a, bank.handle.b, bank.handle.ranks, bank.handle.scales, plan.table)]
        torch.cuda.synchronize()
        with torch.cuda.stream(torch.cuda.Stream()):
            torch.cuda._sleep(SLEEP)
            y = ops.adapter_linear(x, s.packed, bank, plan)
            dx, = torch.autograd.grad(y, x, s.dy)
            y = y.detach()
        del bank, plan
        other = [torch.zeros(n, dtype=torch.uint8, device=DEV) for n in sizes * 3]      # (zeros: all of them adapter 0 of rank 0, if they were read)
        torch.cuda.synchronize()
        assert torch.equal(y, want[0]) and torch.equal(dx, want[1]) and len(other)


@gpu
def test_a_layout_that_ends_half_way_is_finished_before_the_next():
    """The first layout is late on its stream and fails between its copies; the next comes from another stream."""
    s = Site(11)
    bank = s.bank(s.old)
    want = s.step(s.bank(s.new))
    s.step(bank)
    live = bank._live
    put(bank, [w.to(DEV) for w in s.new])

    class Fails:                                         # the copies of `down` are queued, those of `up` raise
        calls = 0

        def __getitem__(self, index):
            Fails.calls += 1
            if Fails.calls == 2:
                raise MemoryError
            return torch.zeros_like(live)[index]         # (other values than the right ones)
    torch.cuda.synchronize()
    bank._live = Fails()
    with torch.cuda.stream(torch.cuda.Stream()):
        torch.cuda._sleep(SLEEP)
        with pytest.raises(MemoryError):
            s.call(bank)
    bank._live = live
    with torch.cuda.stream(torch.cuda.Stream()):
        got = s.step(bank)
    torch.cuda.synchronize()
    assert same(got, want)
