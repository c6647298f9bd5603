"""Products whose weights a row chooses: forms of the calls beside those of test_rows_gpu.py, against the same plain implementations and
with its bounds (check, check_route)."""
import threading

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_rows_gpu import RELU, SILU, act64, check, check_route, gen, grouped_case, i32, offsets_of, randn, run_route  # noqa: E402


@pytest.mark.parametrize("sizes", [[1], [7], [0, 3, 0, 4], [32], [31, 1], [1] * 32, [5, 0, 20, 7], [33], [2] * 17], ids=lambda s: "_".join(map(str, s[:4])))
@pytest.mark.parametrize("gather", [0, 40])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_few_rows_in_e4m3(ctx, sizes, gather, mode):
    """Up to 32 rows take stages of 32 rows: narrow results, some of several tiles per CTA, K of one step and of many turns of the ring."""
    for N, K in ((30, 16), (130, 272), (1030, 640), (4096, 1024), (640, 8192)):
        if len(sizes) * N * K <= 1 << 25:
            grouped_case(ctx, sizes, N, K, gather=gather, fp8=True, mode=mode, act=SILU, alpha=0.5)
    grouped_case(ctx, sizes, 200, 64, gather=gather, fp8=True, mode=mode, pad_a=32, pad_o=3, start=0, shift=1, bias=False)


@pytest.mark.parametrize("mode", [0, 1])
def test_few_rows_in_e4m3_of_wide_results(ctx, mode):
    grouped_case(ctx, [24], 50000, 128, fp8=True, mode=mode, act=RELU)
    grouped_case(ctx, [3, 29], 30000, 64, fp8=True, mode=mode, gather=10)
    grouped_case(ctx, [3, 29], 30000, 64, mode=mode, gather=10)


@pytest.mark.parametrize("rows,cols", [(False, False), (True, False), (False, True)])
@pytest.mark.parametrize("M", [20, 300, 9000])
@pytest.mark.parametrize("gather", [0, 100])
@pytest.mark.parametrize("mode", [0, 1])
def test_e4m3_without_scales(ctx, M, rows, cols, gather, mode):
    import scriptrs_b200 as sb

    g = gen(M)
    G, N, K = 2, 300, 208
    a_rows = gather or M
    a, w = randn(g, a_rows, K).to(torch.float8_e4m3fn), randn(g, G, N, K, std=0.25).to(torch.float8_e4m3fn)
    rs = torch.rand(a_rows, device="cuda", generator=g) + 0.5 if rows else None
    cs = torch.rand(G, N, device="cuda", generator=g) + 0.5 if cols else None
    idx = torch.randint(0, a_rows, (M,), device="cuda", generator=g).int() if gather else torch.arange(M, device="cuda").int()
    sizes = [M // 3, M - M // 3]
    off, out = offsets_of(sizes), torch.zeros(M, N, device="cuda", dtype=torch.float32 if mode else torch.bfloat16)
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), G, M, N, K, d_rows=idx.data_ptr() if gather else 0, a_rows=a_rows,
                    out_mode=mode, fp8=True, d_row_scale=rs.data_ptr() if rows else 0, d_col_scale=cs.data_ptr() if cols else 0)
    ctx.synchronize()
    at = 0
    for e, n in enumerate(sizes):
        pick = idx[at:at + n].long()
        x, we = a.float()[pick].double(), w[e].double()
        f = (rs[pick, None].double() if rows else 1.0) * (cs[e].double() if cols else torch.ones(N, device="cuda", dtype=torch.float64))
        check(out[at:at + n], (x @ we.T) * f, (x.abs() @ we.abs().T) * f, mode != 0)
        at += n


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("normalize", [False, True])
@pytest.mark.parametrize("E", [5, 32, 100, 300])
@pytest.mark.parametrize("T", [90, 700])
def test_route_takes_no_nan_of_either_sign(ctx, T, E, bf16, normalize):
    """NaN of both signs and several payloads beside ordinary logits: never chosen, and no weight of the row changes."""
    dtype, bits = (torch.bfloat16, torch.int16) if bf16 else (torch.float32, torch.int32)
    x = randn(gen(E), T, E).to(dtype)
    odd = [0x7fc0, 0xffc0, 0x7f81, 0xff81, 0xffff, 0x7fff] if bf16 else [0x7fc00000, 0xffc00000, 0x7f800001, 0xff800001, 0xffffffff, 0x7fffffff]
    wrap = 1 << (16 if bf16 else 32)
    raw = x.view(bits)
    for r in range(T):
        for j in range(r % 4):
            v = odd[(r + j) % len(odd)]
            raw[r, (3 * r + 5 * j) % E] = v - wrap if v >= wrap // 2 else v
    raw[8] = odd[1] - wrap  # nothing but negative NaN
    assert bool(x.isnan().any())
    k = min(4, E)
    check_route(run_route(ctx, x, k, normalize), x, k, normalize)


@pytest.mark.parametrize("bf16", [False, True])
def test_route_orders_logits_below_the_normal_range(ctx, bf16):
    dtype = torch.bfloat16 if bf16 else torch.float32
    tiny = torch.finfo(dtype).smallest_normal
    x = (torch.randint(-60, 61, (300, 40), device="cuda", generator=gen(2)).double() * (tiny / 64)).to(dtype)
    assert int((x != 0).sum()) > 10000
    check_route(run_route(ctx, x, 6, True), x, 6, True)


def test_contexts_of_two_threads_at_once(ctx):
    """Each with its context, stream and workspace, first calls included; against the same calls one after the other."""
    import scriptrs_b200 as sb

    M, N, K, r, n, E, k = 3000, 1024, 512, 16, 40, 16, 2
    g = gen(9)
    a, w = randn(g, M, K).bfloat16(), randn(g, E, N, K, std=K ** -0.5).bfloat16()
    down, up = randn(g, n, r, K, std=K ** -0.5).bfloat16(), randn(g, n, N, r, std=0.3).bfloat16()
    who = torch.randint(-1, n, (M,), device="cuda", generator=g).int()
    logits = randn(g, M, E)
    size, need = sb.route_topk_workspace(M, E, k), sb.adapter_gemm_workspace(M, r)

    def buffers():
        i = dict(dtype=torch.int32, device="cuda")
        return [torch.zeros(M, k, **i), torch.zeros(M, k, device="cuda"), torch.zeros(E + 1, **i), torch.zeros(M * k, **i), torch.zeros(M, k, **i),
                torch.zeros(M * k, N, device="cuda").bfloat16(), torch.zeros(M, N, device="cuda"), torch.zeros(M, N, device="cuda").bfloat16(),
                torch.zeros(size, dtype=torch.uint8, device="cuda"), torch.zeros(need, dtype=torch.uint8, device="cuda")]

    def calls(c, b, times):
        for _ in range(times):
            sb.route_topk(c, logits.data_ptr(), *(t.data_ptr() for t in b[:5]), M, E, k, b[8].data_ptr(), size)
            sb.grouped_gemm(c, a.data_ptr(), w.data_ptr(), b[5].data_ptr(), b[2].data_ptr(), E, M * k, N, K, d_rows=b[3].data_ptr(), a_rows=M, act=SILU)
            sb.combine_rows(c, b[5].data_ptr(), b[4].data_ptr(), b[1].data_ptr(), b[6].data_ptr(), M, k, N, M * k, out_mode=1)
            sb.adapter_gemm(c, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), who.data_ptr(), b[7].data_ptr(), n, r, M, N, K, b[9].data_ptr(),
                            need)
        c.synchronize()

    one = buffers()
    torch.cuda.synchronize()
    calls(ctx, one, 1)
    both, failed = [buffers(), buffers()], []
    torch.cuda.synchronize()

    def work(b):
        try:
            c = sb.Context(0)
            calls(c, b, 10)
            c.close()
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(b,)) for b in both]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed
    for b in both:
        for x, y in zip(one[:8], b[:8]):
            assert torch.equal(x, y)


@pytest.mark.parametrize("mode", [0, 1, 2])
@pytest.mark.parametrize("fp8", [False, True])
def test_a_row_has_the_same_bits_in_every_form(ctx, fp8, mode):
    """Few rows and many, in place and through an index, alone and beside other groups."""
    import scriptrs_b200 as sb

    N, K, G, rows = 1030, 1040, 3, 9000
    g = gen(7)
    a, w = randn(g, rows, K), randn(g, G, N, K, std=K ** -0.5)
    rs = torch.rand(rows, device="cuda", generator=g) + 0.5 if fp8 else None
    cs = torch.rand(G, N, device="cuda", generator=g) + 0.5 if fp8 else None
    a, w = (t.to(torch.float8_e4m3fn if fp8 else torch.bfloat16) for t in (a, w))
    bias = randn(g, G, N)

    def run(sizes, idx=None):
        M = sum(sizes)
        out, off = torch.zeros(M, N, device="cuda", dtype=torch.float32 if mode else torch.bfloat16), offsets_of(sizes)
        torch.cuda.synchronize()
        sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), G, M, N, K, d_rows=idx.data_ptr() if idx is not None else 0,
                        a_rows=rows, d_bias=bias.data_ptr(), act=SILU, out_mode=mode, fp8=fp8, d_row_scale=rs.data_ptr() if fp8 else 0,
                        d_col_scale=cs.data_ptr() if fp8 else 0)
        ctx.synchronize()
        return out

    whole = run([0, rows, 0])
    idx = torch.randperm(rows, device="cuda", generator=g).int()
    for n in (1, 20, 32, 33, 130, 700, 3000):
        assert torch.equal(run([0, n, 0]), whole[:n]), n
        assert torch.equal(run([0, n, 0], idx), whole[idx[:n].long()]), n
    assert torch.equal(run([3, 25, 4], idx)[3:28], whole[idx[3:28].long()])
    assert torch.equal(run([300, 2500, 4000], idx)[300:2800], whole[idx[300:2800].long()])
