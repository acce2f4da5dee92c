"""The 8-bit integer product: quantised tokens equal to the rule on whole numbers, products against
the exact integers scaled in 64 bits.

Tolerance of an output: the integer sum's conversion to fp32, the token scale's rounding and two
products (4 half steps of 2^-24, and one more for the residual's sum), then half a step u of the type;
fp16 results below the normal range have an absolute half step of 2^-25.  SiLU: silu(a) moves at most
1.1 da; the fast exponential is off by 2 + 1.2 |a| steps of 2^-23, the quotient by 2, the products by 2."""
import pytest
import torch

from estudiocanciones_b200._lib import HMError

pytestmark = pytest.mark.gpu

DEV = "cuda"
H, BF = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _built():
    from estudiocanciones_b200 import build, kernels
    build.build()
    kernels.read_errors(DEV)
    yield
    assert kernels.read_errors(DEV) == 0, "a kernel reported an error bit"


def rule(x):
    """(q, amax) in 64 bits; torch rounds half to even."""
    d = x.double()
    top = d.abs().amax(-1, keepdim=True)
    return torch.where(top > 0, (d * 127 / torch.where(top > 0, top, torch.ones_like(top))).round(), torch.zeros_like(d)), top


def inputs(M, N, K, dtype=H, seed=0):
    g = torch.Generator().manual_seed(seed + M + 3 * N + 7 * K)
    x = torch.randn(M, K, generator=g) * torch.exp(torch.randn(M, 1, generator=g))
    x[:, ::37] *= 6
    w = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    s = (0.5 + torch.rand(N, generator=g)).mul(1 / (64 * K ** 0.5)).half()
    return x.to(dtype).to(DEV), w.to(DEV), s.to(DEV)


def check(out, x, w, s, res=None, silu=False, rows=slice(None)):
    q, top = rule(x[rows])
    y = (q @ w.double().t()) * (top / 127) * s.double()
    u = torch.finfo(x.dtype).eps / 2
    st = 2.0 ** -24
    if silu:
        a, b = y.chunk(2, -1)
        ref = a * torch.sigmoid(a) * b
        tol = u * ref.abs() + 1.1 * 4 * st * (a * b).abs() + (4 * st + (6 + 1.2 * a.abs()) * 2 * st) * ref.abs()
    else:
        ref = y if res is None else y + res[rows].double()
        tol = u * ref.abs() + 4 * st * y.abs() + st * ref.abs()
    tol = tol * (1 + u) + (2.0 ** -25 if x.dtype == H else 2.0 ** -134)
    d = (out[rows].double() - ref).abs()
    assert bool((d <= tol).all()), f"worst {float((d / tol).max()):.3f} of the tolerance"


# ----------------------------------------------------------------------------- tokens
@pytest.mark.parametrize("M,K,dtype", [(1, 16, H), (3, 48, BF), (7, 4096, H), (300, 272, BF), (2, 16384, H), (2, 20000, BF),
                                       (1, 131072, H)])
def test_tokens(M, K, dtype):
    from estudiocanciones_b200 import kernels
    x, _, _ = inputs(M, 1, K, dtype)
    q, sx = kernels.quant_tokens(x)
    want, top = rule(x)
    assert torch.equal(q.double(), want)
    assert torch.equal(sx, (top[:, 0] / 127).float()), "the quotient's nearest fp32 value"


@pytest.mark.parametrize("dtype", [H, BF])
def test_tokens_at_every_half(dtype):
    """Rows whose quotients are exact halves and their neighbours, at several magnitudes."""
    from estudiocanciones_b200 import kernels
    rows = []
    for top in (127.0, 254.0, 63.5, 1.0, 3.0, 100.0):
        steps = torch.arange(-127, 127).double() + 0.5
        v = (steps * top / 127).to(dtype)
        near = torch.cat([v, (v.float() * (1 + torch.finfo(dtype).eps)).to(dtype), (v.float() * (1 - torch.finfo(dtype).eps)).to(dtype)])
        near = near[near.abs() <= top]
        row = torch.zeros(768, dtype=dtype)
        row[:near.numel()] = near
        row[767] = top
        rows.append(row)
    x = torch.stack(rows).to(DEV)
    lo = torch.finfo(dtype).smallest_normal
    scales = [1.0, 2.0 ** -9, 2.0 ** 6] + ([2.0 ** -120, 2.0 ** -133, 2.0 ** 110] if dtype == BF else [lo])
    for f in scales:
        y = (x.double() * f).to(dtype)
        q, sx = kernels.quant_tokens(y)
        want, top = rule(y)
        assert torch.equal(q.double(), want), f"scale {f}"
        assert torch.equal(sx, (top[:, 0] / 127).float())


def test_tokens_of_the_largest_magnitudes():
    """bf16 rows up to the type's largest value: 127 x leaves the 32-bit range there, the quotients do not."""
    from estudiocanciones_b200 import kernels
    halves = torch.arange(-127, 127).double() + 0.5           # 8 significant bits at most: exact in bf16
    row = torch.cat([halves, torch.tensor([127.0, -127.0]).double()])
    for e in (113, 114, 117, 118, 120, 121):
        x = torch.stack([row * 2.0 ** e, row.flip(0) * 2.0 ** (e - 1)]).bfloat16().to(DEV)
        q, sx = kernels.quant_tokens(x)
        want, top = rule(x)
        assert torch.equal(q.double(), want), f"scale 2^{e}"
        assert torch.equal(sx, (top[:, 0] / 127).float())
    x = (torch.rand(40, 1040, generator=torch.Generator().manual_seed(5)) * 2 - 1).bfloat16()
    x[:, 7] = 1.0
    x = (x.double() * torch.finfo(BF).max).bfloat16().to(DEV)
    q, sx = kernels.quant_tokens(x)
    want, top = rule(x)
    assert torch.equal(q.double(), want) and torch.equal(sx, (top[:, 0] / 127).float())


def test_tokens_zero_and_not_finite():
    from estudiocanciones_b200 import kernels
    x = torch.randn(5, 64, device=DEV).half()
    x[1] = 0
    x[2, 63] = float("inf")
    x[3, 0] = float("nan")
    x[4, 5] = -float("inf")
    w = torch.randint(-127, 128, (40, 64), device=DEV, dtype=torch.int8)
    s = torch.full((40,), 0.01, device=DEV).half()
    q, sx = kernels.quant_tokens(x)
    assert float(sx[1]) == 0 and bool(sx[2:].isnan().all()) and not q[1:].any()
    y = kernels.int8_mm_a8(x, w, s)
    assert bool(y[2:].isnan().all()) and not y[1].any()
    check(y, x, w, s, rows=slice(0, 2))
    z = kernels.int8_mm_a8(x, w, s, silu=True)
    assert bool(z[2:].isnan().all()) and not z[1].any()


# ----------------------------------------------------------------------------- products
@pytest.mark.parametrize("M,N,K,dtype", [
    (1, 1, 16, H), (1, 5, 32, BF), (1, 4096, 2048, H), (2, 8197, 1024, H), (8, 5120, 2048, BF), (9, 100, 144, H),
    (16, 1000, 8192, H), (31, 17, 112, BF), (33, 640, 4096, H), (64, 2304, 512, BF), (127, 129, 1040, H), (128, 128, 128, H),
    (129, 260, 272, BF), (200, 8197, 256, H), (333, 1024, 2048, BF), (257, 4000, 528, H), (700, 3000, 1024, H),
    (1024, 2048, 4096, BF), (513, 5003, 1040, H)])
@pytest.mark.parametrize("res", [False, True])
def test_product(M, N, K, dtype, res):
    from estudiocanciones_b200 import kernels
    x, w, s = inputs(M, N, K, dtype)
    r = torch.randn(M, N, device=DEV).to(dtype) if res else None
    check(kernels.int8_mm_a8(x, w, s, r), x, w, s, r)


@pytest.mark.parametrize("M,N,K,dtype", [
    (1, 2, 16, H), (1, 16384, 1024, H), (3, 30, 64, BF), (8, 16384, 2048, H), (16, 2 * 1000, 512, BF), (40, 2 * 72, 1040, H),
    (128, 2 * 2048, 1024, H), (150, 2 * 501, 256, BF), (300, 2 * 4096, 512, H), (1000, 2 * 2500, 1040, BF)])
def test_product_with_silu(M, N, K, dtype):
    from estudiocanciones_b200 import kernels
    x, w, s = inputs(M, N, K, dtype)
    check(kernels.int8_mm_a8(x, w, s, silu=True), x, w, s, silu=True)


@pytest.mark.parametrize("M,N", [(3, 64), (300, 5000)])
def test_product_of_the_largest_magnitudes(M, N):
    """bf16 rows near the type's largest value: the integer sum times the token's scale leaves the 32-bit range,
    the result does not."""
    from estudiocanciones_b200 import kernels
    x, w, s = inputs(M, N, 272, BF)
    x = (x / x.abs().amax(-1, keepdim=True) * 2.0 ** 126).to(BF)
    s = (s.float() * 2.0 ** -14 / s.float().max()).half()
    y = kernels.int8_mm_a8(x, w, s)
    assert bool(y.isfinite().all())
    check(y, x, w, s)


@pytest.mark.parametrize("M,F", [(2, 40), (300, 5000)])
def test_silu_of_far_negative_values(M, F):
    """bf16 with a between -91 and -80, where silu(a) still is a normal number and b is large.

    Tolerance, relative: a's conversion, scale and two products move a by 4 half steps, so a e^a by 4 (1 + |a|) of them, b by 4;
    the exponential is off by 4 + 1.2 |a| steps of 2^-23, the quotient by 2, four products by half a step each; then half a
    step of the type."""
    from estudiocanciones_b200 import kernels
    x = torch.zeros(M, 16, device=DEV, dtype=BF)
    x[:, 3] = 1.0
    w = torch.zeros(2 * F, 16, device=DEV, dtype=torch.int8)
    w[:F, 3], w[F:, 3] = -127, 127
    s = torch.cat([torch.linspace(80 / 127, 91 / 127, F), torch.full((F,), 60000.0)]).half().to(DEV)
    y = kernels.int8_mm_a8(x, w, s, silu=True).double()
    a, b = -127 * s[:F].double(), 127 * s[F:].double()
    ref = (a * torch.sigmoid(a) * b).expand(M, F)
    tol = torch.finfo(BF).eps / 2 + (4 * (1 + a.abs()) + 4 + 2 * (4 + 1.2 * a.abs()) + 4 + 4) * 1.01 * 2.0 ** -24
    d = (y - ref).abs() / ref.abs()
    assert bool((d <= tol).all()), f"worst {float((d / tol).max()):.3f} of the tolerance"


def test_the_longest_sums():
    """K = 131072 with every product at its largest: the sum 127 * 127 * K is held exactly."""
    from estudiocanciones_b200 import kernels
    K = 131072
    x = torch.ones(3, K, device=DEV).half()
    x[1] = -1
    w = torch.full((9, K), 127, dtype=torch.int8, device=DEV)
    w[4, 5:] = -127
    s = torch.full((9,), 2.0 ** -12, device=DEV).half()
    check(kernels.int8_mm_a8(x, w, s), x, w, s)


def test_large_activation_offsets():
    """Rows whose element offsets pass 2^31."""
    from estudiocanciones_b200 import kernels
    M, K, N = 18000, 131072, 8
    x = torch.zeros(M, K, device=DEV, dtype=H)
    x[-3:] = torch.randn(3, K, device=DEV).half()
    w = torch.randint(-127, 128, (N, K), device=DEV, dtype=torch.int8)
    s = torch.full((N,), 2.0 ** -12, device=DEV).half()
    y = kernels.int8_mm_a8(x, w, s)
    assert not y[:-3].any()
    check(y, x, w, s, rows=slice(M - 3, M))


@pytest.mark.parametrize("M", [5, 600])
def test_parts_strides_and_in_place(M):
    """quant_tokens + gemm_i8a8 == int8_mm_a8; row pitches; odd offsets; out == res; leading dimensions."""
    from estudiocanciones_b200 import kernels
    N, K = 1000, 512
    x, w, s = inputs(M, N, K)
    want = kernels.int8_mm_a8(x, w, s)
    q, sx = kernels.quant_tokens(x)
    assert torch.equal(kernels.gemm_i8a8(q, sx, w, s), want)
    wide = torch.zeros(M, K + 64, device=DEV, dtype=torch.int8)
    wide[:, 16:16 + K] = q
    assert torch.equal(kernels.gemm_i8a8(wide[:, 16:16 + K], sx, w, s), want)
    for off in (8, 3):                                      # rows on 16 bytes, and not (copied)
        buf = torch.randn(M, K + 24, device=DEV).half()
        buf[:, off:off + K] = x
        assert torch.equal(kernels.int8_mm_a8(buf[:, off:off + K], w, s), want)
    for off, pad in ((8, 16), (1, 5), (3, 8)):              # vector stores, and element ones
        out = torch.full((M, N + pad + 8), 9.0, device=DEV).half()
        kernels.int8_mm_a8(x, w, s, out=out[:, off:off + N])
        assert torch.equal(out[:, off:off + N], want)
        assert bool((out[:, :off] == 9).all()) and bool((out[:, off + N:] == 9).all())
    r = torch.randn(M, N, device=DEV).half()
    both = kernels.int8_mm_a8(x, w, s, r)
    buf = r.clone()
    assert kernels.int8_mm_a8(x, w, s, buf, out=buf) is buf and torch.equal(buf, both)
    rw = torch.zeros(M, N + 3, device=DEV).half()
    rw[:, 1:1 + N] = r
    assert torch.equal(kernels.int8_mm_a8(x, w, s, rw[:, 1:1 + N]), both)
    y = kernels.int8_mm_a8(x.view(M, 1, K), w, s, r.view(M, 1, N))
    assert y.shape == (M, 1, N) and torch.equal(y.view(M, N), both)
    assert torch.equal(kernels.int8_mm_a8(x[0], w, s), want[0])


def test_rows_do_not_depend_on_their_number():
    """The integers are exact, so a row's result is the same in a call of 1 and of 1000 rows."""
    from estudiocanciones_b200 import kernels
    x, w, s = inputs(1000, 2 * 1536, 1024)
    for silu in (False, True):
        all_rows = kernels.int8_mm_a8(x, w, s, silu=silu)
        for m in (1, 7, 100, 130, 513):
            assert torch.equal(kernels.int8_mm_a8(x[:m], w, s, silu=silu), all_rows[:m])


def test_streams_and_graphs():
    from estudiocanciones_b200 import kernels
    from estudiocanciones_b200._lib import capture_graph
    x, w, s = inputs(40, 640, 512)
    want = kernels.int8_mm_a8(x, w, s)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        ys = [kernels.int8_mm_a8(x, w, s) for _ in range(5)]
    here = [kernels.int8_mm_a8(x, w, s) for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in ys + here)
    g, cs = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    x2, w2 = x.clone(), w.clone()
    with capture_graph(g, cs):
        w2.copy_(w2.flip(0))                                # the weights are made just before the call
        y = kernels.int8_mm_a8(x2, w2, s)
        z = kernels.int8_mm_a8(y[:, :512], w2, s)           # and a call reads the last one's result
    w2.copy_(w)
    for i in range(4):
        x2.copy_(x.roll(i, 0))
        g.replay()
        check(y, x2, w2, s)
        check(z, y[:, :512].contiguous(), w2, s)
    del g


def test_refused_arguments():
    from estudiocanciones_b200 import kernels
    x, w, s = inputs(4, 64, 128)
    q, sx = kernels.quant_tokens(x)
    r = torch.zeros(4, 64, device=DEV).half()
    for f in (lambda: kernels.int8_mm_a8(x.float(), w, s), lambda: kernels.int8_mm_a8(x[:, :120], w[:, :120], s),
              lambda: kernels.int8_mm_a8(x, w[:, :64], s), lambda: kernels.int8_mm_a8(x, w[:, ::2], s),
              lambda: kernels.int8_mm_a8(x, w, s.float()), lambda: kernels.int8_mm_a8(x, w, s[:-1]),
              lambda: kernels.int8_mm_a8(x, w.t(), s), lambda: kernels.int8_mm_a8(x, w, s, r.bfloat16()),
              lambda: kernels.int8_mm_a8(x, w, s, r[:, :32]), lambda: kernels.int8_mm_a8(x, w, s, r, silu=True),
              lambda: kernels.int8_mm_a8(x, w[:63], s[:63], silu=True), lambda: kernels.int8_mm_a8(x, w, s, out=r[:3]),
              lambda: kernels.int8_mm_a8(x, w, s, out=r.t()), lambda: kernels.int8_mm_a8(x[:0], w, s),
              lambda: kernels.int8_mm_a8(x.cpu(), w, s), lambda: kernels.int8_mm_a8(x, w.cpu(), s),
              lambda: kernels.quant_tokens(x[:, :8]), lambda: kernels.quant_tokens(q),
              lambda: kernels.quant_tokens(torch.zeros(1, 131088, device=DEV).half()),
              lambda: kernels.gemm_i8a8(q, sx.half(), w, s), lambda: kernels.gemm_i8a8(q, sx[:3], w, s),
              lambda: kernels.gemm_i8a8(x, sx, w, s), lambda: kernels.gemm_i8a8(q, sx, w, s, dtype=torch.float32),
              lambda: kernels.gemm_i8a8(q.t(), sx, w, s)):
        with pytest.raises(HMError):
            f()
