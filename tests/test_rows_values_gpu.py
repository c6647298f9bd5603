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
