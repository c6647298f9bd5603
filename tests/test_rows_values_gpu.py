"""Products whose weights a row chooses, through the C ABI: values whose relative error, not only their error against the sum of
absolute products, is known beforehand."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

SILU = 1


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------------------------------------------------------- SiLU
def silu_check(out, x, mode):
    """out [M, N] against silu(x), x [N] f32, given exactly to the activation.
    Of the 32-bit function's own: exp's argument is off by |x| 2^-23 at most (product and constant), exp, quotient, sum and product by a
    few 2^-22.  Below 2^-100 the exponential leaves the normal range: an absolute bound."""
    ref = x.double() * torch.sigmoid(x.double())
    own = 2.0 ** -20 + x.double().abs() * 2.0 ** -23
    bound = ((1.0 + 2.0 ** -8) * (1.0 + own) - 1.0 if mode == 0 else own) * ref.abs() + 2.0 ** -100
    assert torch.isfinite(out).all()
    far = (out.double() - ref).abs()
    worst = (far / ref.abs().clamp(min=2.0 ** -100)).amax(0)
    assert bool((far <= bound).all()), (float(worst.max()), float(x[worst.argmax()]))


def pre_activations(n):
    x = torch.linspace(-24.0, 12.0, n, device="cuda")
    x[::17] *= 5.0  # down to -120: the exponential of the other sign would overflow
    x[n // 3] = 0.0
    return x


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("gather", [0, 40])
@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("M,N", [(1, 30), (20, 1024), (200, 1030), (9000, 1024)])
def test_silu_of_a_grouped_product(ctx, M, N, gather, mode, fp8):
    """Weights of zero: the bias alone is what the activation gets.  Few rows, tiles of every kind, narrow columns."""
    import scriptrs_b200 as sb

    K, G = 16, 2
    dt = torch.float8_e4m3fn if fp8 else torch.bfloat16
    a_rows = gather or M
    a, w = torch.ones(a_rows, K, device="cuda").to(dt), torch.zeros(G, N, K, device="cuda").to(dt)
    x = pre_activations(N)
    bias = torch.stack([x, x])
    rows = (torch.arange(M, device="cuda") % a_rows).int() if gather else None
    out = torch.zeros(M, N, device="cuda", dtype=torch.float32 if mode else torch.bfloat16)
    off = i32([0, M // 3, M])
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), G, M, N, K, d_rows=rows.data_ptr() if gather else 0, a_rows=a_rows,
                    d_bias=bias.data_ptr(), act=SILU, out_mode=mode, fp8=fp8)
    ctx.synchronize()
    silu_check(out, x, mode)


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("M", [5, 33, 9000])
def test_silu_beside_adapters(ctx, M, mode):
    import scriptrs_b200 as sb

    N, K, r = 1024, 16, 8
    a, w = torch.ones(M, K, device="cuda").bfloat16(), torch.zeros(N, K, device="cuda").bfloat16()
    down, up = torch.zeros(2, r, K, device="cuda").bfloat16(), torch.ones(2, N, r, device="cuda").bfloat16()
    x = pre_activations(N)
    who = (torch.arange(M, device="cuda") % 3 - 1).int()
    out = torch.zeros(M, N, device="cuda", dtype=torch.float32 if mode else torch.bfloat16)
    size = sb.adapter_gemm_workspace(M, r)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    sb.adapter_gemm(ctx, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), who.data_ptr(), out.data_ptr(), 2, r, M, N, K, work.data_ptr(), size,
                    d_bias=x.data_ptr(), act=SILU, out_mode=mode)
    ctx.synchronize()
    silu_check(out, x, mode)


# ------------------------------------------------------------------------------------------------------------ adapters
def adapters_alone(ctx, a, down, up, who, mode):
    """The addition by itself, beside shared weights of zero."""
    import scriptrs_b200 as sb

    (M, K), (n, N, r) = a.shape, up.shape
    w = torch.zeros(N, K, device="cuda").bfloat16()
    out = torch.full((M, N), 3.0, device="cuda", dtype=torch.float32 if mode else torch.bfloat16)
    size = sb.adapter_gemm_workspace(M, r)
    work = torch.full((size,), 0xff, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    sb.adapter_gemm(ctx, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), who.data_ptr(), out.data_ptr(), n, r, M, N, K, work.data_ptr(), size,
                    out_mode=mode)
    ctx.synchronize()
    return out


FORMS = [1, 32, 33, 200, 2500, 9000]  # rows: CUDA cores, then tiles of 128 rows and of 256


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("M", FORMS)
@pytest.mark.parametrize("rank", [8, 24])
def test_an_addition_that_cancels(ctx, M, rank, mode):
    """low = (257, 256, 0, ...) against up = (c, -c, 0, ...): c, where 257 in bf16 would give 0 or 2 c.  The values are exact in bf16."""
    K, N = 16, 1024
    a = torch.ones(M, K, device="cuda").bfloat16()
    down, up = torch.zeros(2, rank, K, device="cuda").bfloat16(), torch.zeros(2, N, rank, device="cuda").bfloat16()
    down[:, 0, 0], down[:, 0, 1], down[:, 1, 0] = 256.0, 1.0, 256.0
    c = (torch.arange(N, device="cuda") % 19 - 9).float()
    up[:, :, 0], up[:, :, 1] = c.bfloat16(), -c.bfloat16()
    who = (torch.arange(M, device="cuda") // 3 % 2).int()
    out = adapters_alone(ctx, a, down, up, who, mode)
    assert torch.equal(out.float(), c.expand(M, N))


@pytest.mark.parametrize("rank", [8, 64, 128])
def test_a_row_keeps_its_numbers_whatever_the_batch(ctx, rank):
    """`low` enters with an error of 2^-16 of |low| |up| at most (two bf16 terms), is itself summed in 32 bits (K / 16 MMAs, 17 addends cut
    off at 2^-23 each: below 2^-16 of |x| |down| |up|), and the result is rounded once: 2^-8.  So the same row differs by a rounding to
    bf16 at most between a call of 32 rows and one of 33 or more."""
    K, N, n = 64, 512, 4
    g = torch.Generator(device="cuda").manual_seed(rank)
    a = torch.randn(max(FORMS), K, device="cuda", generator=g).bfloat16()
    down = (torch.randn(n, rank, K, device="cuda", generator=g) * K ** -0.5).bfloat16()
    up = (torch.randn(n, N, rank, device="cuda", generator=g) * rank ** -0.5).bfloat16()
    who = torch.randint(-1, n, (max(FORMS),), device="cuda", generator=g).int()
    ref = torch.zeros(max(FORMS), N, device="cuda", dtype=torch.float64)
    size = torch.zeros_like(ref)
    for e in range(n):
        here = who == e
        low = a[here].double() @ down[e].double().T
        ref[here] = low @ up[e].double().T
        size[here] = (low.abs() + a[here].double().abs() @ down[e].double().abs().T) @ up[e].double().abs().T
    bound = 2.0 ** -16 * size + (1.0 + 2.0 ** -7) * 2.0 ** -8 * ref.abs()
    few = None
    for M in FORMS:
        out = adapters_alone(ctx, a[:M], down, up, who[:M].contiguous(), 0).double()
        far = (out - ref[:M]).abs()
        assert bool((far <= bound[:M]).all()), (M, float((far - bound[:M]).max()))
        if M == 32:
            few = out
        elif few is not None:
            assert bool(((out[:32] - few).abs() <= 2.0 ** -15 * size[:32] + (1.0 + 2.0 ** -7) * 2.0 ** -7 * few.abs()).all()), M


# -------------------------------------------------------------------------------------------------- sums in 32 bits
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("M,gather", [(20, 0), (200, 0), (200, 50), (20000, 0)])
@pytest.mark.parametrize("K", [512, 1024, 4096])
def test_small_products_beside_a_large_one(ctx, K, M, gather, fp8):
    """The tensor core cuts addends off where they reach below the largest one's 24 bits and some bits more; a 32-bit result is collected every
    512 columns of K.  So of one product of 2^16 with small positive ones beside it no more is lost than what 511 of them have below
    2^-16 of it: 511 x 2^-25 of the sum for three bits more (measured: 112 x 2^-23), whatever K and the type."""
    import scriptrs_b200 as sb

    N, a_rows = 128, gather or M
    dt = torch.float8_e4m3fn if fp8 else torch.bfloat16
    off, rows = i32([0, M]), (torch.arange(M, device="cuda") % a_rows).int()
    for e in range(-16, -3):
        a, w = torch.full((a_rows, K), 2.0 ** (e // 2), device="cuda"), torch.full((N, K), 1.75 * 2.0 ** (e - e // 2), device="cuda")
        a[:, 0] = w[:, 0] = 256.0
        a, w = a.to(dt), w.to(dt)
        ref = (a[:1].double() @ w.double().T)[0]
        out = torch.zeros(M, N, device="cuda")
        torch.cuda.synchronize()
        sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), 1, M, N, K, d_rows=rows.data_ptr() if gather else 0, a_rows=a_rows,
                        out_mode=1, fp8=fp8)
        ctx.synchronize()
        far = float(((out.double() - ref).abs() / ref).max())
        assert far <= 128 * 2.0 ** -23, (e, far * 2 ** 23)
