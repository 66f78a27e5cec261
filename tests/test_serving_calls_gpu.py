"""How the operators of the batched decode step are called: devices, streams, gradients."""
import threading
import time

import pytest

import tmac_zynq_fpga_b200 as tm
from test_serving import append, cache, draw
from test_serving_gpu import BF16, append_case, check_append

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu


def test_a_refused_device_leaves_nothing_behind():
    """The refusal is the call's alone: the next launch does not report it."""
    for device in (99, -1):
        assert draw(device=device) == -9 and append(cache(device=device)) == -9
        check_append(append_case(BF16, BF16, 14, 2, 64, 64, 16, 5))
        torch.zeros(3, device="cuda").add_(1)


def busy_stream():
    """A stream that is some tenths of a second behind."""
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)
    return side


@pytest.mark.parametrize("by_address", [False, True])
@pytest.mark.parametrize("which", ["rope_append", "prefix_attention", "sample"])
def test_arguments_dropped_after_a_call_on_another_stream(which, by_address):
    """torch must not give their memory to the next tensor while that stream has yet to read it."""
    c = append_case(BF16, BF16, 14, 2, 64, 64, 16, 64, n_seq=64)
    cache = tm.PagedCache(*c["pools"])
    inputs = {"rope_append": c["q"].contiguous(), "prefix_attention": c["q"].contiguous(), "sample": torch.randn(64, 5000, device="cuda")}[which]
    lens, u = c["pos"] - c["starts"] + 1, torch.full((64,), 0.5, device="cuda")

    def call(x, **kw):
        if which == "rope_append":
            return tm.rope_append(cache, x, c["k"], c["v"], c["pos"], c["tables"], c["cos"], c["sin"], starts=c["starts"], **kw)
        if which == "prefix_attention":
            return tm.prefix_attention(x, cache, c["tables"], lens, **kw)
        return tm.sample(x, u, **kw)[0]

    tm.rope_append(cache, c["q"], c["k"], c["v"], c["pos"], c["tables"], c["cos"], c["sin"], starts=c["starts"])
    want = call(inputs)
    temporary = inputs.clone()
    torch.cuda.synchronize()
    side = busy_stream()
    got = call(temporary, stream=side.cuda_stream if by_address else side)
    del temporary
    later = [torch.full_like(inputs, -7.0) for _ in range(4)]
    side.synchronize()
    assert torch.equal(got, want) and len(later) == 4


def test_a_tensor_that_requires_grad_is_refused():
    """The operators have no gradient: a result without history would train nothing, silently."""
    c = append_case(BF16, BF16, 14, 2, 64, 64, 16, 6, n_seq=6)
    lens = c["pos"] - c["starts"] + 1
    x = dict(q=c["q"].contiguous(), k=c["k"].contiguous(), v=c["v"].contiguous(), bias=c["bias"], cos=c["cos"], sin=c["sin"], kp=c["pools"][0],
             vp=c["pools"][1], logits=torch.randn(6, 100, device="cuda"), t=torch.ones(6, device="cuda"))

    def call(which, **kw):
        d = {**x, **kw}
        cache = tm.PagedCache(d["kp"], d["vp"])
        if which == "append":
            return tm.rope_append(cache, d["q"], d["k"], d["v"], c["pos"], c["tables"], d["cos"], d["sin"], starts=c["starts"], bias=d["bias"])
        if which == "attention":
            return tm.prefix_attention(d["q"], cache, c["tables"], lens)
        return tm.sample(d["logits"], torch.zeros(6, device="cuda"), temperature=d["t"])[0]

    for which, names in (("append", ["q", "k", "v", "bias", "cos", "sin", "kp", "vp"]), ("attention", ["q", "kp", "vp"]), ("sample", ["logits", "t"])):
        want = call(which)
        for name in names:
            grad = {name: x[name].clone().requires_grad_()}
            with pytest.raises(tm.TmacError, match="grad"):
                call(which, **grad)
            with torch.no_grad():
                assert torch.equal(call(which, **grad), want)
            assert torch.equal(call(which, **{name: grad[name].detach()}), want)


@pytest.mark.parametrize("which", ["rope_append", "prefix_attention", "sample"])
def test_other_threads_run_while_a_launch_waits(which):
    """A stream that takes no more launches holds up the thread that launches, not the interpreter."""
    c = append_case(BF16, BF16, 2, 1, 64, 64, 16, 2, n_seq=2)
    cache = tm.PagedCache(*c["pools"])
    logits, u, lens = torch.zeros(2, 100, device="cuda"), torch.zeros(2, device="cuda"), c["pos"] - c["starts"] + 1
    q = torch.zeros(2, 2, 64, dtype=BF16, device="cuda")

    def call():
        if which == "rope_append":
            tm.rope_append(cache, c["q"], c["k"], c["v"], c["pos"], c["tables"], c["cos"], c["sin"], starts=c["starts"], q_out=q)
        elif which == "prefix_attention":
            tm.prefix_attention(q, cache, c["tables"], lens, out=q)
        else:
            tm.sample(logits, u)

    call()
    torch.cuda._sleep(1000)
    torch.cuda.synchronize()
    ticks, done = [time.perf_counter()], threading.Event()

    def tick():
        while not done.is_set():
            time.sleep(0.002)
            ticks.append(time.perf_counter())

    other = threading.Thread(target=tick)
    side = torch.cuda.Stream()
    other.start()
    t0 = time.perf_counter()
    with torch.cuda.stream(side):
        torch.cuda._sleep(3_000_000_000)
        for _ in range(4000):
            call()
    queued = time.perf_counter() - t0
    done.set()
    other.join()
    side.synchronize()
    longest = max(b - a for a, b in zip(ticks, ticks[1:]))
    assert queued > 1.0  # the queue was full for most of the stream's sleep
    assert longest < queued / 2
