"""Linear layer with bias, activation and residual in its epilogue: refusals
and the feed-forward on the CPU, the gfx950 kernels against formulas in 64 bits."""

import math

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from replay_amd.ops.fused_linear import fused_linear

requires_gpu = pytest.mark.skipif(not torch.cuda.is_available(), reason="needs ROCm GPU")
ACTS = ["none", "relu", "gelu", "silu"]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def activation(z, act):
    """act(z), its slope, and a bound of the slope's own slope."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).double(), 0.0
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        pdf = torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
        return z * cdf, cdf + z * pdf, 0.8  # |2 phi(z) - z^2 phi(z)| <= 2 phi(0)
    if act == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s), 0.5
    return z, torch.ones_like(z), 0.0


def make(M, K, N, dtype, bias=True, residual=True, seed=0):
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=gen) * scale).to(dtype).cuda()

    x, w = normal(M, K), normal(N, K, scale=1 / math.sqrt(max(K, 1)))
    return x, w, normal(N) if bias else None, normal(M, N) if residual else None, normal(M, N)


def check(x, w, b, r, dy, act, dtype):
    """Outputs and gradients, each within what its roundings allow.

    Half a step h of the type (2^-24 for float32).  z is a float32 sum of K + 1
    terms: off by (K + 2) 2^-24 of their absolute sum Z.  |slope| <= 1.2, and
    the activations' own float32 functions are good to 2^-21.  The slope is
    taken at z rounded to the type: off by (its own slope's bound) x (h |z| +
    z's error); dz is rounded to the type once for the two products, and their
    float32 sums are off by (terms + 2) 2^-24 of the absolute sum."""
    h, f = torch.finfo(dtype).eps / 2, 2.0**-24
    (M, K), N = x.shape, w.shape[0]
    leaves = [t.detach().requires_grad_() for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, w, b, r)]
    y = fused_linear(args[0], args[1], args[2], activation=act, residual=args[3])
    grads = torch.autograd.grad(y, leaves, dy)
    assert y.dtype == dtype and all(g.dtype == dtype for g in grads)
    xd, wd, dyd = x.double(), w.double(), dy.double()
    z = xd @ wd.t()
    Z = xd.abs() @ wd.abs().t()
    if b is not None:
        z, Z = z + b.double(), Z + b.double().abs()
    a, slope, curve = activation(z, act)
    out = a if r is None else a + r.double()
    # below fp16's normal range a rounding is a fixed step
    floor = 2.0**-25 if dtype == torch.float16 else 1e-37
    z_off = (K + 2) * f * Z
    y_off = 1.2 * z_off + 2.0**-21 * a.abs() + 2 * f * out.abs()
    got = dict(y=(y.detach(), out, y_off * (1 + h) + h * out.abs() + floor))
    # relu's slope jumps where z is not told from 0: there dz may be all or nothing
    slope_off = curve * (h * z.abs() + z_off + floor) + 2.0**-21
    if act == "relu":
        slope_off = slope_off + (z.abs() <= z_off + floor).double()
    dz = dyd * slope
    dz_off = dyd.abs() * slope_off
    rounded = dz_off + (h * (dz.abs() + dz_off) + floor if act != "none" else 0.0)
    whole = dz.abs() + rounded
    tol = {
        "dx": rounded @ wd.abs() + (N + 2) * f * (whole @ wd.abs()),
        "dw": rounded.t() @ xd.abs() + (M + 2) * f * (whole.t() @ xd.abs()),
        "db": rounded.sum(0) + (M + 2) * f * whole.sum(0),
        "dr": torch.zeros_like(dyd),
    }
    exact = {"dx": dz @ wd, "dw": dz.t() @ xd, "db": dz.sum(0), "dr": dyd}
    names = [n for n, t in zip(("dx", "dw", "db", "dr"), (x, w, b, r)) if t is not None]
    for name, g in zip(names, grads):
        got[name] = (g, exact[name], tol[name] * (1 + h) + h * exact[name].abs() + (0 if name == "dr" else floor))
    for name, (value, want, bound) in got.items():
        assert value.shape == want.shape, name
        assert torch.isfinite(value).all(), name
        off = (value.double() - want).abs()
        assert not (off > bound).any(), f"{name}: off by {off.max():.3e}, {float((off / bound).max()):.2f} times"


class TestCpu:
    @pytest.mark.parametrize("act", ACTS)
    def test_gradients_against_differences(self, act):
        gen = torch.Generator().manual_seed(0)

        def leaf(*shape):
            return torch.randn(*shape, generator=gen, dtype=torch.float64).requires_grad_()

        args = (leaf(2, 3, 4), leaf(5, 4), leaf(5), leaf(2, 3, 5))
        assert torch.autograd.gradcheck(lambda x, w, b, r: fused_linear(x, w, b, act, r), args)

    def test_refusals(self):
        x, w, b, r = torch.zeros(2, 3, 4), torch.zeros(5, 4), torch.zeros(5), torch.zeros(2, 3, 5)
        for bad in (
            dict(activation="tanh"),
            dict(weight=torch.zeros(4, 5)),
            dict(weight=torch.zeros(4)),
            dict(weight=w.double()),
            dict(bias=torch.zeros(4)),
            dict(bias=torch.zeros(1, 5)),
            dict(residual=torch.zeros(3, 5)),  # never broadcast
            dict(residual=torch.zeros(2, 3, 4)),
            dict(residual=r.half()),
        ):
            with pytest.raises(ValueError):
                fused_linear(**{**dict(x=x, weight=w, bias=b, residual=r), **bad})
        with pytest.raises(ValueError, match="dtype"):
            fused_linear(x.int(), w.int())

    @pytest.mark.parametrize("act", ["relu", "gelu"])
    def test_feed_forward_is_the_same(self, act):
        from replay_amd.nn import PointWiseFeedForward

        torch.manual_seed(0)
        plain = PointWiseFeedForward(8, 0.3, act, hidden_dim=12)
        fused = PointWiseFeedForward(8, 0.3, act, hidden_dim=12, fused=True)
        fused.load_state_dict(plain.state_dict())
        x = torch.randn(3, 5, 8)
        for mode in (True, False):
            torch.manual_seed(1)
            want = plain.train(mode)(x)
            torch.manual_seed(1)
            torch.testing.assert_close(fused.train(mode)(x), want)


@pytest.mark.gpu
@requires_gpu
class TestKernels:
    @pytest.mark.parametrize("dtype", DTYPES, ids=str)
    @pytest.mark.parametrize("act", ACTS)
    @pytest.mark.parametrize("residual", [False, True])
    @pytest.mark.parametrize("M,K,N", [(200, 64, 64), (65, 256, 96)])
    def test_activations(self, M, K, N, act, residual, dtype):
        check(*make(M, K, N, dtype, residual=residual), act, dtype)

    @pytest.mark.parametrize("dtype", DTYPES, ids=str)
    @pytest.mark.parametrize(
        "M,K,N",
        [
            (1, 1, 1), (1, 64, 200), (3, 7, 5), (16, 32, 16), (17, 33, 31), (64, 64, 64), (127, 129, 65),
            (300, 1000, 40), (1000, 8, 1030), (5000, 64, 192), (8, 256, 1024), (70, 2048, 136), (257, 520, 264),
        ],
    )
    @pytest.mark.parametrize("bias", [False, True])
    def test_sizes(self, M, K, N, bias, dtype):
        check(*make(M, K, N, dtype, bias=bias, residual=bias), "gelu" if bias else "none", dtype)

    @pytest.mark.parametrize("dtype", DTYPES, ids=str)
    def test_strides(self, dtype):
        # rows of a wider buffer, off 16-byte alignment; a transposed weight; a broadcast gradient
        gen = torch.Generator().manual_seed(0)
        x = torch.randn(100, 71, generator=gen).to(dtype).cuda()[:, 1:66]
        w = (torch.randn(65, 48, generator=gen) / 8).to(dtype).cuda().t()
        r = torch.randn(100, 50, generator=gen).to(dtype).cuda()[:, :48]
        b = torch.randn(96, generator=gen).to(dtype).cuda()[::2]
        dy = torch.ones((), dtype=dtype, device="cuda").expand(100, 48)
        check(x, w, b, r, dy, "silu", dtype)

    @pytest.mark.parametrize("dtype", DTYPES, ids=str)
    def test_leading_dimensions_and_nothing(self, dtype):
        x, w, b, _, _ = make(24, 16, 40, dtype, residual=False)
        flat = fused_linear(x, w, b, "relu")
        assert torch.equal(fused_linear(x.view(2, 3, 4, 16), w, b, "relu"), flat.view(2, 3, 4, 40))
        assert fused_linear(x[0], w, b, "relu").shape == (40,)
        for M, K, N in ((0, 4, 5), (3, 0, 5), (3, 4, 0)):
            check(*make(M, K, N, dtype), "gelu", dtype)

    def test_refusals(self):
        x, w, b, r, _ = make(6, 4, 5, torch.float32)
        fused_linear(x, w, b, "relu", r)
        for change in (
            dict(weight=w.cpu()), dict(weight=w.half()), dict(weight=w[:, :3]), dict(weight=w[0]),
            dict(bias=b[:4]), dict(bias=b[None]), dict(bias=b.cpu()), dict(residual=r[:1]), dict(residual=r[:, :4]),
            dict(residual=r.half()), dict(residual=r.cpu()), dict(x=x.double()), dict(x=x[0, 0]),
            dict(x=x.double(), weight=w.double(), bias=b.double(), residual=r.double()), dict(activation="tanh"),
        ):
            for grad in (False, True):
                args = {**dict(x=x, weight=w, bias=b, residual=r, activation="none"), **change}
                args["x"] = args["x"].detach().requires_grad_(grad)
                with pytest.raises(ValueError):
                    fused_linear(**args)

    def test_far_offsets(self):
        # rows that end past 2^31 elements, and outputs past 2^32 bytes
        gen = torch.Generator().manual_seed(0)
        store = torch.empty(2**31 + 2**22, dtype=torch.bfloat16, device="cuda")
        M, K, stride = 2049, 64, 2**20
        x = store.as_strided((M, K), (stride, 1)).copy_(torch.randn(M, K, generator=gen))
        w, b = (torch.randn(48, K, generator=gen) / 8).bfloat16().cuda(), torch.randn(48, generator=gen).bfloat16().cuda()
        dy = torch.randn(M, 48, generator=gen).bfloat16().cuda()
        leaves, near = [[t.detach().requires_grad_() for t in (a, w, b)] for a in (x, x.contiguous())]
        for args in zip(
            torch.autograd.grad(fused_linear(*leaves, "gelu"), leaves, dy),
            torch.autograd.grad(fused_linear(*near, "gelu"), near, dy),
        ):
            assert torch.equal(*args)
        tall = torch.randn(2**25 + 3, 8, device="cuda").bfloat16()
        wide = torch.randn(72, 8, device="cuda").bfloat16()
        y = fused_linear(tall, wide)
        assert torch.equal(y[-300:], fused_linear(tall[-300:], wide))

    def test_two_graphs_in_turn(self):
        cases = [make(3000, 64, 128, torch.bfloat16, seed=i) for i in (1, 2)]
        graphs, held = [], []

        def step(x, w, b, r, dy):
            return torch.autograd.grad(fused_linear(x, w, b, "gelu", r), [x, w, b], dy)

        for case in cases:
            for t in case[:3]:
                t.requires_grad_()
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step(*case)
            torch.cuda.current_stream().wait_stream(side)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
                held.append(step(*case))
            graphs.append(graph)
        for _ in range(3):
            for i, case in enumerate(cases):
                graphs[i].replay()
                got = [t.clone() for t in held[i]]
                for a, c in zip(got, step(*case)):
                    assert torch.equal(a, c)

    def test_backward_twice(self):
        x, w, b, r, dy = make(300, 64, 48, torch.bfloat16)
        leaves = [t.requires_grad_() for t in (x, w, b, r)]
        y = fused_linear(x, w, b, "silu", r)
        first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        for a, c in zip(first, torch.autograd.grad(y, leaves, dy)):
            assert torch.equal(a, c)

    def test_large_values(self):
        # far beyond where exp overflows, both ways
        x = torch.tensor([[1000.0], [-1000.0], [88.0], [-88.0], [-104.0], [0.0]], device="cuda")
        w = torch.ones(1, 1, device="cuda")
        for act in ACTS:
            check(x, w, None, None, torch.ones(6, 1, device="cuda"), act, torch.float32)

    @pytest.mark.parametrize("act", ACTS)
    def test_nan_and_infinity_pass(self, act):
        x = torch.tensor([[math.nan], [math.inf], [1.0]], device="cuda")
        y = fused_linear(x, torch.ones(1, 1, device="cuda"), activation=act)
        assert torch.isnan(y[0]).all() and torch.isinf(y[1]).all() and torch.isfinite(y[2]).all()

    def test_gradient_at_nan_is_torchs(self):
        x = torch.tensor([[math.nan], [-1.0], [0.0], [2.0]], device="cuda")
        w = torch.ones(1, 1, device="cuda")
        grads = []
        for f in (lambda t: fused_linear(t, w, activation="relu"), lambda t: torch.relu(t @ w.t())):
            leaf = x.clone().requires_grad_()
            grads.append(torch.autograd.grad(f(leaf).sum(), leaf)[0])
        assert torch.equal(*grads)

    def test_same_bits_again(self):
        x, w, b, r, dy = make(20000, 64, 64, torch.bfloat16)
        leaves = [t.requires_grad_() for t in (x, w, b)]

        def grads():
            return torch.autograd.grad(fused_linear(x, w, b, "gelu", r), leaves, dy)

        for g, again in zip(grads(), grads()):
            assert torch.equal(g, again)

    def test_frozen_inputs(self):
        x, w, b, r, dy = make(100, 32, 48, torch.bfloat16)
        for wanted in ((x,), (w,), (b,), (r,), (x, b)):
            for t in (x, w, b, r):
                t.requires_grad_(False)
            for t in wanted:
                t.requires_grad_()
            got = torch.autograd.grad(fused_linear(x, w, b, "silu", r), wanted, dy)
            for t in (x, w, b, r):
                t.requires_grad_()
            full = dict(zip("xwbr", torch.autograd.grad(fused_linear(x, w, b, "silu", r), (x, w, b, r), dy)))
            for g, t in zip(got, wanted):
                name = "xwbr"[[t is u for u in (x, w, b, r)].index(True)]
                assert torch.equal(g, full[name])

    def test_autocast(self):
        x, w, b, r, dy = make(100, 32, 48, torch.float32)
        w.requires_grad_()
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = fused_linear(x, w, b, "gelu", r)
        assert y.dtype == torch.bfloat16
        (dw,) = torch.autograd.grad(y, [w], dy.bfloat16())
        assert dw.dtype == torch.float32
        with torch.no_grad():
            assert torch.equal(y, fused_linear(*(t.bfloat16() for t in (x, w, b)), "gelu", r.bfloat16()))

    def test_another_stream_and_graph(self):
        x, w, b, r, dy = make(3000, 64, 128, torch.bfloat16)
        leaves = [t.requires_grad_() for t in (x, w, b)]

        def step():
            y = fused_linear(x, w, b, "gelu", r)
            return (y.detach(), *torch.autograd.grad(y, leaves, dy))

        want = step()
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        for a, c in zip(got, want):
            assert torch.equal(a, c)
        del got
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for seed in (5, 6, 7):
            with torch.no_grad():
                x.copy_(make(3000, 64, 128, torch.bfloat16, seed=seed)[0])
            graph.replay()
            want = step()
            torch.cuda.synchronize()
            for a, c in zip(held, want):
                assert torch.equal(a, c)


@pytest.mark.gpu
@requires_gpu
class TestForwardModeAndTraces:
    """What the kernels cannot carry is refused, and a trace holds the call."""

    @pytest.mark.parametrize("which", range(4))
    @pytest.mark.parametrize("grad", [False, True])
    def test_tangents(self, which, grad):
        args = list(make(8, 4, 5, torch.float32)[:4])
        args[0].requires_grad_(grad)
        with forward_ad.dual_level():
            args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises(RuntimeError):
                fused_linear(*args[:3], residual=args[3])

    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
    def test_trace(self, dtype):
        x, w, b, r, _ = make(70, 40, 24, dtype)

        def call(x, r):
            return fused_linear(x, w, b, "gelu", r)

        with torch.no_grad():
            traced = torch.jit.trace(call, (x, r), check_trace=False)
            assert torch.equal(traced(2 * x, 3 * r), call(2 * x, 3 * r))


class TestFeedForwardOnCpu:
    def test_dropout_kept_on_in_serving(self):
        """Dropout switched on by itself, as for an estimate of uncertainty."""
        from replay_amd.nn import PointWiseFeedForward

        torch.manual_seed(0)
        plain = PointWiseFeedForward(8, 0.5)
        fused = PointWiseFeedForward(8, 0.5, fused=True)
        fused.load_state_dict(plain.state_dict())
        x = torch.randn(3, 5, 8)
        for name in ("dropout1", "dropout2"):
            outs = []
            for module in (plain, fused):
                module.eval()
                getattr(module, name).train()
                torch.manual_seed(1)
                outs.append(module(x))
            torch.testing.assert_close(*outs)


@pytest.mark.gpu
@requires_gpu
class TestAutocastOnGpu:
    @pytest.mark.parametrize("dtype", [torch.float64, torch.int32], ids=str)
    @pytest.mark.parametrize("grad", [False, True])
    def test_leaves_other_types_alone(self, dtype, grad):
        x, w = torch.ones(6, 4, device="cuda"), torch.ones(5, 4, device="cuda", requires_grad=grad)
        b, r = torch.ones(5, device="cuda"), torch.ones(6, 5, device="cuda")
        with torch.autocast("cuda", dtype=torch.bfloat16):
            fused_linear(x, w, b, residual=r)
            for bad in (
                (x.to(dtype), w, b, r), (x, w.detach().to(dtype), b, r), (x, w, b.to(dtype), r), (x, w, b, r.to(dtype)),
                tuple(t.detach().to(dtype) for t in (x, w, b, r)),
            ):
                with pytest.raises(ValueError):
                    fused_linear(*bad[:3], residual=bad[3])


class TestAutocastOnCpu:
    def test_casts_as_on_the_gpu(self):
        gen = torch.Generator().manual_seed(0)
        x, w, b, r = (torch.randn(*s, generator=gen) for s in ((6, 4), (5, 4), (5,), (6, 5)))
        w.requires_grad_()
        with torch.autocast("cpu", dtype=torch.bfloat16):
            y = fused_linear(x.bfloat16(), w, b, "gelu", r)  # mixed types, as a stack of layers has them
            z = fused_linear(x.double(), w.detach().double(), b.double())
        assert y.dtype == torch.bfloat16 and z.dtype == torch.float64
        assert torch.equal(y, fused_linear(*(t.bfloat16() for t in (x, w, b)), "gelu", r.bfloat16()))
        (dw,) = torch.autograd.grad(y.sum(), [w])
        assert dw.dtype == torch.float32


@pytest.mark.gpu
@requires_gpu
class TestTiles:
    """Each tile of each product, with ragged edges: (rows, K, N), and what the
    forward product, dx and dW (in how many parts of the rows) run on."""

    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
    @pytest.mark.parametrize("act", ["none", "gelu"])
    @pytest.mark.parametrize(
        "M,K,N",
        [
            (4097, 1032, 4104),  # 256x256; 128x128; 128x128 in 4 waves, 1 part
            (4097, 4104, 1032),  # 128x128; 256x256; as above
            (33000, 136, 72),    # 128x64, two stages; the same; 128x128 in 8 waves, 104 parts
            (33001, 56, 48),     # 128x64, one stage; the same; 64x64, 104 parts
            (4097, 1031, 4103),  # 128x128 through registers; 64x64 so; 64x64 so, 1 part
            (4097, 4103, 1031),  # 64x64 so; 128x128 so; as above
            (2001, 1416, 1504),  # 128x64, two stages; the same; 128x128 in 4 waves, 3 parts
            (2000, 136, 72),     # 64x64; the same; 128x128 in 8 waves, 7 parts
        ],
    )
    def test_16_bits(self, M, K, N, act, dtype):
        check(*make(M, K, N, dtype, residual=act != "none"), act, dtype)

    @pytest.mark.parametrize(
        "M,K,N",
        [
            (4097, 516, 4100),  # 128x128; 128x64, two stages; 128x128, 3 parts
            (4097, 4100, 516),  # 128x64, two stages; 128x128; 128x128, 3 parts
            (33000, 68, 72),    # 128x64, two stages; the same; 128x128, 104 parts
            (33001, 32, 64),    # 128x64, one stage; two stages; 64x64, 104 parts
            (4097, 515, 4099),  # 64x64 through registers
        ],
    )
    def test_float32(self, M, K, N):
        check(*make(M, K, N, torch.float32), "silu", torch.float32)

    @pytest.mark.parametrize("off", [8, 3])
    def test_rows_of_a_wider_buffer(self, off):
        # 256x256 with whole chunks, and through registers off 16 bytes
        gen = torch.Generator().manual_seed(0)
        M, K, N = 4097, 1032, 4104
        x = torch.randn(M, K + 16, generator=gen).bfloat16().cuda()[:, off : off + K]
        w = (torch.randn(N, K + 8, generator=gen) / 32).bfloat16().cuda()[:, :K]
        r = torch.randn(M, N + 24, generator=gen).bfloat16().cuda()[:, off : off + N]
        b = torch.randn(N, generator=gen).bfloat16().cuda()
        dy = torch.randn(M, N + 8, generator=gen).bfloat16().cuda()[:, :N]
        check(x, w, b, r, dy, "relu", torch.bfloat16)
