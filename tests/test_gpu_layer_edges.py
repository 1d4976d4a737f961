"""The layer operators at the edges of their range: the bounds are those of
test_gpu_layer.py unless a test derives its own."""
import pytest
import torch

from ferrograd_b200 import kernels
from test_gpu_layer import forward_case, grad_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k,xl", [(17, 4999, 4096, "plain"), (20, 2501, 4096, "plain"),
                                      (68, 5001, 4096, "plain"), (122, 5001, 8192, "plain"),
                                      (43, 4999, 4096, "transposed")])
def test_few_rows_into_an_odd_width(dtype, m, n, k, xl):
    """Wide split tiles whose rows leave through slabs: the most shared memory."""
    forward_case(dtype, m, n, k, "relu", None, False, True, False, m, xl)


def test_gradient_of_few_rows_and_an_odd_width():
    grad_case("bf16", 20, 4096, 2501, "none", None, 1)


# ---- streams: the allocator's blocks are ordered on the stream they belong to ----------


DELAY = 200_000_000  # cycles, about a tenth of a second


def one_of_each(stream):
    """A call of each operator on a given stream, by name."""
    gen = torch.Generator(device="cuda").manual_seed(1)
    new = lambda r, c: torch.empty((r, c), device="cuda").normal_(generator=gen)  # noqa: E731
    x, w, dy, pre = new(1024, 512), new(1024, 512), new(1024, 1024), new(1024, 1024)
    torch.cuda.synchronize()
    drop = kernels.Dropout(0.25, 3, 4)
    return {
        "linear": lambda: kernels.linear(x, w, act="silu", drop=drop, save_pre=True, stream=stream),
        "linear_grad": lambda: kernels.linear_grad(dy, x, w, pre=pre, act="silu", drop=drop,
                                                   stream=stream),
        "dropout": lambda: (kernels.dropout(dy, drop, stream=stream),),
    }


@pytest.mark.parametrize("name", ["linear", "linear_grad", "dropout"])
def test_given_stream_leaves_the_current_ones_memory_alone(name):
    """A block freed on the current stream with work on it still to run: neither
    does that work reach the call's results, nor the call that work's input."""
    side = torch.cuda.Stream()
    call = one_of_each(side.cuda_stream)[name]
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    for _ in range(2):  # the results of 4 MB, then the workspaces of 3 to 13
        torch.cuda.empty_cache()
        later = torch.empty_like(want[0])
        early = [torch.full((n << 18,), 5.0, device="cuda") for n in (1, 3, 4, 6, 13)]
        copies = [torch.empty_like(t) for t in early]
        torch.cuda.synchronize()
        torch.cuda._sleep(DELAY)
        later.fill_(7)
        for c, t in zip(copies, early):
            c.copy_(t)
        del later, early, t
        got = call()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
        for c in copies:
            assert bool((c == 5).all())


@pytest.mark.parametrize("name", ["linear", "linear_grad", "dropout"])
def test_given_stream_keeps_what_the_call_still_uses(name):
    """The call waits on its stream; results and arguments dropped meanwhile are not
    handed to the current stream before it is done with them."""
    side = torch.cuda.Stream()
    calls = one_of_each(side.cuda_stream)
    want = [t.clone() for t in calls[name]()]
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    calls = one_of_each(side.cuda_stream)
    with torch.cuda.stream(side):
        torch.cuda._sleep(DELAY)
    got = calls[name]()
    if name != "dropout":  # the last result is not wanted: pre, or db
        sizes = [got[-1].numel()]
        got = got[:-1]
    else:
        sizes = []
    del calls  # nor are the arguments kept
    others = [torch.zeros(n, device="cuda")
              for n in sizes + [1 << 19, 1 << 19, 1 << 20, 1 << 20] for _ in range(2)]
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for z in others:
        assert not z.any()


@pytest.mark.parametrize("explicit", [False, True])
def test_two_streams_at_once(explicit):
    """Calls with workspaces on two streams in turn, with no wait between them."""
    gen = torch.Generator(device="cuda").manual_seed(2)
    cases = []
    for dt, m, n, k in ((torch.float32, 300, 500, 700), (torch.bfloat16, 257, 333, 1001),
                        (torch.float16, 64, 1030, 2047), (torch.float32, 40, 96, 2050)):
        new = lambda r, c: torch.empty((r, c), dtype=dt, device="cuda").normal_(  # noqa: E731
            generator=gen)
        cases.append((new(m, k), new(n, k) / 32, new(m, n), new(m, n)))
    drop = kernels.Dropout(0.1, 5, 6)

    def calls(x, w, dy, pre, stream=None):
        out, z = kernels.linear(x, w, act="gelu", residual=dy, drop=drop, save_pre=True,
                                stream=stream)
        return (out, z, kernels.dropout(dy, drop, stream=stream)) + kernels.linear_grad(
            dy, x, w, pre=pre, act="gelu", drop=drop, stream=stream)

    want = [calls(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(40):
        c = cases[i * 3 % 4]
        if explicit:
            got.append((i * 3 % 4, calls(*c, stream=streams[i % 2].cuda_stream)))
        else:
            with torch.cuda.stream(streams[i % 2]):
                got.append((i * 3 % 4, calls(*c)))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(r, want[i]))
