"""The layer operators at the edges of their range: the bounds are those of
test_gpu_layer.py unless a test derives its own."""
import ctypes
import threading

import numpy as np
import pytest
import torch

from ferrograd_b200 import CudaDevice, kernels
from ferrograd_b200.device import Event
from layer_ref import act as ref_act, linear_grad as ref_grad, slope as ref_slope
from test_gpu_layer import CURVE, ROUND, STEP, TINY, TYPES, check, f64, forward_case, grad_case, \
    randn

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
    want = call()
    torch.cuda.synchronize()
    want = [t.clone() for t in want]
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
    want = calls[name]()
    torch.cuda.synchronize()
    want = [t.clone() for t in want]
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


# ---- infinities and overflow in f32 ------------------------------------------------------


ROWS = [(5, 40, 72), (40, 96, 200), (300, 264, 136), (2560, 2304, 96)]


def same_class(got, ref, what):
    """Equal infinities and NaN; finite where the definition is."""
    got = f64(got)
    for of in (np.isnan, np.isposinf, np.isneginf):
        assert np.array_equal(of(got), of(ref)), (what, of.__name__)


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("m,n,k", ROWS)
def test_f32_infinities_are_f32s(m, n, k, act):
    """Infinities of both signs in x and in w, zeros opposite some, and two
    opposite each other: every element is what the 64-bit formula gives."""
    rng = np.random.default_rng(m)
    x, w, dy = (randn(rng, *s, torch.float32) for s in ((m, k), (n, k), (m, n)))
    x[1, 5], x[m - 1, 7], w[2, 9], w[n - 1, 5] = np.inf, -np.inf, -np.inf, np.inf
    w[3, 5] = w[4, 7] = x[0, 9] = 0.0
    x[2, 11] = x[2, 12] = np.inf
    w[6, 11], w[6, 12] = 1.0, -1.0
    with np.errstate(invalid="ignore"):
        z = f64(x) @ f64(w).T
        same_class(kernels.linear(x, w, act=act), ref_act(z, act), "out")
        dy[1, 3], dy[3, 3] = np.inf, -np.inf
        got = kernels.linear_grad(dy, x, w)
        for g, r, name in zip(got, (f64(dy) @ f64(w), f64(dy).T @ f64(x), f64(dy).sum(0)),
                              ("dx", "dw", "db")):
            same_class(g, r, name)


@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("m,n,k", ROWS)
def test_f32_overflow_keeps_its_sign(m, n, k, act):
    """Finite operands whose products are beyond f32: infinite, of the sum's sign.
    In each row of x the terms are of one sign, so no order of summation gives
    NaN; the last column is small enough to stay finite."""
    rng = np.random.default_rng(n)
    for big_x, big_w in ((1.5e21, 1.5e21), (3e38, 3.9), (3e38, 40.0), (1e30, 1e9)):
        x = torch.from_numpy(rng.uniform(0.5, 1.0, (m, k)) * big_x).float().cuda()
        w = torch.from_numpy(rng.uniform(0.5, 1.0, (n, k)) * big_w).float().cuda()
        x[1::2] *= -1
        w[n - 1] = torch.from_numpy(rng.uniform(0.0, 1e-3 / k, k)).float()
        z = f64(x) @ f64(w).T
        z[np.abs(z) > 3.5e38] *= np.inf
        assert np.isinf(z[:, :n - 1]).all() and np.isfinite(z[:, n - 1]).all()
        same_class(kernels.linear(x, w, act=act), ref_act(z, act), (big_x, big_w))


# ---- dz in 16 bits -----------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("act", ["none", "relu"])
@pytest.mark.parametrize("m,n,k", [(90, 72, 56), (300, 512, 264), (2560, 2304, 320)])
def test_grad_without_a_slope_is_rounded_once(dtype, act, m, n, k):
    """Dropout's scale 1/(1 - p) is no 16-bit value; the products see dy all the
    same.  One rounding of normally distributed values to bf16 is off by 0.85 2^-9
    in the 2-norm (f16: 2^-12), two in a row by 1.2; between them lies the bound
    for dx and dw.  db, of fewer values, is held to the largest error."""
    gen = torch.Generator(device="cuda").manual_seed(m)
    dt = TYPES[dtype]
    new = lambda r, c, s=1.0: torch.empty((r, c), dtype=dt, device="cuda").normal_(  # noqa: E731
        0, s, generator=gen)
    dy, x, w, pre = new(m, n), new(m, k), new(n, k, 0.1), new(m, n)
    spec = (0.3, 3, 1 << 40)
    got = kernels.linear_grad(dy, x, w, pre=pre, act=act, drop=kernels.Dropout(*spec))
    dx, dw, db, dz = ref_grad(f64(dy), f64(x), f64(w), f64(pre), act, spec)
    for g, r, most in zip(got, (dx, dw, db), (0.5, 0.5, 1.0)):
        assert np.linalg.norm(f64(g) - r) <= most * ROUND[dtype] * np.linalg.norm(r)


@pytest.mark.parametrize("act,at", [("none", 0.0), ("relu", 1.0), ("gelu", 1.4), ("gelu_tanh", 1.4),
                                    ("silu", 2.4)])
@pytest.mark.parametrize("m,n,k", [(40, 64, 72), (300, 264, 136), (2560, 2304, 96)])
def test_f16_grad_beyond_f16s_range(act, at, m, n, k):
    """dz is up to 1.13 * 65504 / (1 - p), the gradients are not: no infinity.
    The bounds are grad_case's; a slope near its maximum."""
    rng = np.random.default_rng(m + n)
    spec = (0.5, 5, 6) if m != 300 else None
    dy = torch.from_numpy(rng.choice([-65504.0, 65504.0, 60000.0], (m, n))).half().cuda()
    x, w = randn(rng, m, k, torch.float16, 1e-3), randn(rng, n, k, torch.float16, 1e-3)
    pre = torch.full((m, n), at, dtype=torch.float16, device="cuda")
    got = kernels.linear_grad(dy, x, w, pre=pre, act=act, need_db=False,
                              drop=kernels.Dropout(*spec) if spec else None)
    dx, dw, _, dz = ref_grad(f64(dy), f64(x), f64(w), f64(pre), act, spec)
    u, tiny = ROUND["f16"], TINY["f16"]
    r = (CURVE * 2 + 2 * STEP + u) * np.abs(dz)
    for g, ref, left, right, terms, rr in ((got[0], dx, np.abs(dz), np.abs(f64(w)), n, r),
                                           (got[1], dw, np.abs(dz).T, np.abs(f64(x)), m, r.T)):
        assert np.abs(ref).max() < 65504
        check(g, ref, (terms + 16) * STEP * (left @ right) + rr @ right + u * np.abs(ref) + tiny,
              act)


# ---- the activations' tails ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [3, 2000])
def test_left_tails_keep_their_digits(dtype, act, rows):
    """act and its slope for z in [-8, -1.5], through w = 1, relative to their
    value.  Phi by its polynomial is good to 2^-15.  An exponential's argument is at
    most 49 (the tanh form's at -8) and three times rounded, 2^-24 each: 2^-16.8 of
    the value; f32's functions add little, so 2^-16.5 there and 2^-14 in 16 bits.
    The slopes are differences that shrink by at most 5 (SiLU's zero is at -1.28):
    2^-14 and 2^-11.5.  Then the output's rounding; f16 adds one unit among
    subnormals to each rounding, of which the slope has two, the first of a half."""
    z = torch.linspace(-8, -1.5, rows, device="cuda").to(TYPES[dtype]).view(-1, 1)
    one = torch.ones((1, 1), dtype=TYPES[dtype], device="cuda")
    near, steep = (2.0 ** -16.5, 2.0 ** -14) if dtype == "f32" else (2.0 ** -14, 2.0 ** -11.5)
    ref = ref_act(f64(z), act)
    check(kernels.linear(z, one, act=act), ref, (near + ROUND[dtype]) * np.abs(ref) + TINY[dtype],
          act)
    ref = ref_slope(f64(z), act)
    dx = kernels.linear_grad(torch.ones_like(z), z, one, pre=z, act=act)[0]
    check(dx, ref, (steep + 2 * ROUND[dtype]) * np.abs(ref) + 2 * TINY[dtype], act)


# ---- the bias gradient's sums ----------------------------------------------------------------


@pytest.mark.parametrize("m,n,most", [(256, 128, -23.0), (8192, 4096, -23.0), (100000, 64, -22.5),
                                      (16, 1100000, -23.0)])
def test_f32_bias_gradient_is_summed_as_a_tree(m, n, most):
    """Random terms: a rounding has 0.18 of 2^-48 of its partial sum's variance.
    In a chain of c roundings the partial sums average half of the whole, in a
    tree's level they are all of it: at most 16 / 2 rows a thread, 6 levels (3 in
    large arrays) and the last rounding make 1.6 2^-24 at most; 100000 rows are
    joined from 782 blocks, 25 compensated additions a thread (one rounding) and 5
    levels more, 1.9 2^-24.  A chain of 128 would add 11 to the variance."""
    gen = torch.Generator(device="cuda").manual_seed(n)
    dy = torch.empty((m, n), device="cuda").normal_(generator=gen)
    x, w = torch.zeros((m, 1), device="cuda"), torch.zeros((n, 1), device="cuda")
    db = kernels.linear_grad(dy, x, w, need_dx=False, need_dw=False)[2]
    ref = dy.double().sum(0)
    assert float((db - ref).norm() / ref.norm()) <= 2.0 ** most
    again = kernels.linear_grad(dy, x, w, need_dx=False, need_dw=False)[2]
    assert torch.equal(db, again)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_bias_gradient_of_the_longest_batch(dtype):
    """2^31 - 256 rows: the last block of rows ends where an int does."""
    m = 0x7fffff00
    dy = torch.zeros((m, 1), dtype=TYPES[dtype], device="cuda")
    for at in (0, m // 2, m - 1):
        dy[at] = 1.0
    one = torch.ones((1, 1), dtype=TYPES[dtype], device="cuda")
    db = kernels.linear_grad(dy, one.expand(m, 1), one, need_dx=False, need_dw=False)[2]
    assert float(db) == 3.0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", [(5, 8), (70, 33)])
def test_no_outputs_leave_the_gradient_that_went_round(dtype, m, k):
    """N = 0: dx is dx_residual, whatever its rows' stride (repeated, overlapping, wide)."""
    dt = TYPES[dtype]
    new = lambda *s: torch.empty(s, dtype=dt, device="cuda").normal_()  # noqa: E731
    dy, x, w = new(m, 0), new(m, k), new(0, k)
    for r in (new(1, k).expand(m, k), new(m + k).as_strided((m, k), (1, 1)), new(m, k + 3)[:, 2:2 + k],
              new(m, k)):
        dx, dw, db = kernels.linear_grad(dy, x, w, dx_residual=r)
        assert torch.equal(dx, r) and dw.shape == (0, k) and db.shape == (0,)
    assert not kernels.linear_grad(dy, x, w)[0].any()


def test_a_failed_call_leaves_no_error_behind():
    """The runtime's last error after a refused call is not there for torch's next
    launch to find (two events that were never recorded have no time between)."""
    device = CudaDevice()
    start, end = Event(device), Event(device)
    with pytest.raises(kernels._lib.FerroError):
        Event.elapsed_ms(start, end)
    assert float((torch.ones(8, device="cuda") + 1).sum()) == 16


# ---- what the binding refuses or passes on ---------------------------------------------------


def test_lazily_negated_views_are_refused():
    """The imaginary part of a conjugate shares memory that holds its negative."""
    z = torch.randn((6, 6), device="cuda", dtype=torch.complex64).conj().imag
    assert z.is_neg()
    w = torch.randn((6, 6), device="cuda")
    for call in (lambda t: kernels.linear(t, w), lambda t: kernels.linear(w, t),
                 lambda t: kernels.linear(w, w, residual=t), lambda t: kernels.linear(w, w, out=t),
                 lambda t: kernels.linear_grad(t, w, w), lambda t: kernels.linear_grad(w, w, t),
                 lambda t: kernels.dropout(t, kernels.Dropout(0.5, 1))):
        with pytest.raises(ValueError):
            call(z)
        call(z.resolve_neg())


def test_out_of_memory_is_torchs():
    """Outputs of 8 TB: the allocator refuses before anything is launched."""
    one = torch.ones((1, 1), dtype=torch.bfloat16, device="cuda")
    x, w = one.expand(1 << 21, 1), one.expand(1 << 21, 1)
    with pytest.raises(torch.OutOfMemoryError):
        kernels.linear(x, w)
    with pytest.raises(torch.OutOfMemoryError):
        kernels.dropout(torch.ones((1, 1 << 21), dtype=torch.bfloat16, device="cuda")
                        .expand(1 << 21, 1 << 21), None)
    assert float(kernels.linear(one, one)) == 1.0


@pytest.mark.parametrize("dtype", TYPES)
def test_a_new_threads_first_call(dtype):
    """A thread that has made no CUDA call yet has no context bound to it."""
    dt = TYPES[dtype]
    x, w = torch.randn((300, 264), device="cuda").to(dt), torch.randn((136, 264), device="cuda").to(dt)
    dy = torch.randn((300, 136), device="cuda").to(dt)
    calls = [lambda: kernels.linear(x, w), lambda: kernels.linear_grad(dy, x, w)[0],
             lambda: kernels.linear(x[:1], w), lambda: kernels.dropout(x, kernels.Dropout(0.5, 1))]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    for call, ref in zip(calls, want):
        got = []
        thread = threading.Thread(target=lambda: got.append(call()))
        thread.start()
        thread.join()
        torch.cuda.synchronize()
        assert got and torch.equal(got[0], ref)


def test_threads_call_at_once():
    """The C entry point from eight threads, each with its stream and buffers (ctypes
    lets go of the interpreter's lock), the first calls of their kernels among them."""
    L = kernels._lib.lib()
    shapes = [(200, 136, 264, torch.float32), (64, 72, 2048, torch.float16),
              (40, 8200, 512, torch.bfloat16), (2600, 2312, 96, torch.float32)]
    codes = {torch.float32: kernels._lib.F32, torch.bfloat16: kernels._lib.BF16,
             torch.float16: kernels._lib.F16}
    jobs = []
    for i in range(8):
        m, n, k, dt = shapes[i % 4]
        x, w = torch.randn((m, k), device="cuda").to(dt), torch.randn((n, k), device="cuda").to(dt)
        out, ws = torch.zeros((m, n), dtype=dt, device="cuda"), torch.empty(1 << 26, dtype=torch.uint8,
                                                                           device="cuda")
        a = kernels._lib.LinearArgsC(dtype=codes[dt], M=m, N=n, K=k, x=x.data_ptr(), x_row=k, x_col=1,
                                     w=w.data_ptr(), w_row=k, w_col=1, out=out.data_ptr(), ld_out=n,
                                     workspace=ws.data_ptr(), workspace_bytes=ws.numel())
        jobs.append((a, torch.cuda.Stream(), x, w, out, ws))
    torch.cuda.synchronize()
    start, failed, done = threading.Barrier(8), [], []

    def work(a, stream):
        start.wait()
        for _ in range(50):
            if L.fg_linear(ctypes.byref(a), stream.cuda_stream):
                failed.append(L.fg_last_error())
        done.append(1)

    threads = [threading.Thread(target=work, args=job[:2]) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert len(done) == 8 and not failed, failed[:1]
    for a, _, x, w, out, _ in jobs:
        assert torch.equal(out, kernels.linear(x, w))


# ---- long sums of one sign -------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("m,n,k", [(256, 512, 16384), (2560, 2304, 16384), (256, 512, 60000)])
def test_long_sums_hardly_drift(dtype, m, n, k):
    """The tensor cores cut each addition of 16 products, by up to 2^-22 of the sum
    so far.  Over a chain of c additions of one sign the sums average half of the
    last one: c 2^-23 of it; f16 takes chains of 256 (2^-15), bf16 of 1024 (2^-13), which
    are added without drift.  The mean signed error of many outputs, spread over two
    binades, shows that: the roundings, to nearest, average out (2^-9.3 / sqrt(2^17)
    in bf16)."""
    gen = torch.Generator(device="cuda").manual_seed(k)
    new = lambda r, c, lo, hi: torch.empty((r, c), device="cuda").uniform_(  # noqa: E731
        lo, hi, generator=gen)
    x = (new(m, k, 0, 1) * new(m, 1, 0.25, 1)).to(TYPES[dtype])
    w = (new(n, k, 0, 1) / 64).to(TYPES[dtype])
    got = kernels.linear(x, w)
    ref = x.double() @ w.double().t()
    mean = float(((got.double() - ref) / ref).mean())
    assert abs(mean) <= (2.0 ** -13 if dtype == "bf16" else 2.0 ** -15)


# ---- nothing is written beside an output ------------------------------------------------------


GUARD = -77.0


def guarded(rows, cols, dt, pitch):
    """[rows, cols] inside a buffer of GUARD, and a check that the rest still is."""
    buf = torch.full((rows, pitch), GUARD, dtype=dt, device="cuda")

    def intact():
        return bool((buf[:, cols:] == GUARD).all())

    return buf[:, :cols], intact


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [3, 40, 300, 2560])
@pytest.mark.parametrize("less", range(9))
def test_columns_beside_the_outputs_stay(dtype, m, less):
    """Outputs that are the first columns of wider, aligned rows: every width modulo 8,
    in every form of the product.  What lies beside them is somebody else's."""
    dt, L, k, n = TYPES[dtype], kernels._lib.lib(), 72, 2304 - less
    code = {"f32": kernels._lib.F32, "bf16": kernels._lib.BF16, "f16": kernels._lib.F16}[dtype]
    stream = torch.cuda.current_stream().cuda_stream
    new = lambda r, c: torch.randn((r, c), device="cuda").to(dt)  # noqa: E731
    ws = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    x, w, r = new(m, k), new(n, k), new(m, 2320)[:, :n]
    (out, out_ok), (pre, pre_ok) = guarded(m, n, dt, 2320), guarded(m, n, dt, 2336)
    a = kernels._lib.LinearArgsC(
        dtype=code, M=m, N=n, K=k, x=x.data_ptr(), x_row=k, x_col=1, w=w.data_ptr(), w_row=k, w_col=1,
        residual=r.data_ptr(), ld_residual=2320, act=kernels._lib.ACT_RELU, pre=pre.data_ptr(),
        ld_pre=2336, out=out.data_ptr(), ld_out=2320, workspace=ws.data_ptr(),
        workspace_bytes=ws.numel())
    assert L.fg_linear(ctypes.byref(a), stream) == 0
    want = kernels.linear(x, w, act="relu", residual=r, save_pre=True)
    assert torch.equal(out, want[0]) and torch.equal(pre, want[1])
    assert out_ok() and pre_ok()
    # dx [m, n] and dw [k, n] of a layer with n inputs
    x, w, dy = new(m, n), new(k, n), new(m, k)
    (dx, dx_ok), (dw, dw_ok) = guarded(m, n, dt, 2320), guarded(k, n, dt, 2320)
    g = kernels._lib.LinearGradArgsC(
        dtype=code, M=m, N=k, K=n, dy=dy.data_ptr(), dy_row=k, dy_col=1, x=x.data_ptr(), x_row=n,
        x_col=1, w=w.data_ptr(), w_row=n, w_col=1, dx_residual=r.data_ptr(), ld_dx_residual=2320,
        dx=dx.data_ptr(), ld_dx=2320, dw=dw.data_ptr(), ld_dw=2320, workspace=ws.data_ptr(),
        workspace_bytes=ws.numel())
    assert L.fg_linear_grad(ctypes.byref(g), stream) == 0
    want = kernels.linear_grad(dy, x, w, dx_residual=r, need_db=False)
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    assert dx_ok() and dw_ok()
    y, y_ok = guarded(m, n, dt, 2320)
    kernels.dropout(r, kernels.Dropout(0.5, 1), out=y)
    assert y_ok()


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_gradients_leave_the_columns_beside_them(dtype):
    """dw in the pair form too."""
    dt, L = TYPES[dtype], kernels._lib.lib()
    code = {"f32": kernels._lib.F32, "bf16": kernels._lib.BF16, "f16": kernels._lib.F16}[dtype]
    m, n, k = 128, 2560, 2301
    new = lambda r, c: torch.randn((r, c), device="cuda").to(dt)  # noqa: E731
    dy, x, w = new(m, n), new(m, k), new(n, k)
    ws = torch.empty(1 << 28, dtype=torch.uint8, device="cuda")
    dw, ok = guarded(n, k, dt, 2304)
    g = kernels._lib.LinearGradArgsC(
        dtype=code, M=m, N=n, K=k, dy=dy.data_ptr(), dy_row=n, dy_col=1, x=x.data_ptr(), x_row=k,
        x_col=1, w=w.data_ptr(), w_row=k, w_col=1, dw=dw.data_ptr(), ld_dw=2304,
        workspace=ws.data_ptr(), workspace_bytes=ws.numel())
    assert L.fg_linear_grad(ctypes.byref(g), torch.cuda.current_stream().cuda_stream) == 0
    assert torch.equal(dw, kernels.linear_grad(dy, x, w, need_dx=False, need_db=False)[1])
    assert ok()
