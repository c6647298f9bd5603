"""Row products, router and weighted sum on arrays of more than 2^31 elements: rows looked at are spread over the whole, the last ones among
them.  Bounds as in test_rows_gpu.py."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from test_rows_gpu import check, gen, i32, randn  # noqa: E402


@pytest.fixture(autouse=True)
def memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def picks(M, n=200):
    return torch.cat([torch.arange(0, M, M // n, device="cuda"), torch.arange(M - 40, M, device="cuda")])


@pytest.mark.parametrize("mode", [0, 1])
@pytest.mark.parametrize("gather", [False, True])
def test_a_long_result(ctx, gather, mode):
    import scriptrs_b200 as sb

    M, N, K, G = 540003, 4096, 64, 3
    g = gen(1)
    a_rows = 5000 if gather else M
    a, w = randn(g, a_rows, K).bfloat16(), randn(g, G, N, K, std=K ** -0.5).bfloat16()
    rows = torch.randint(0, a_rows, (M,), device="cuda", generator=g).int()
    off = i32([0, 200001, 200001, M])
    out = torch.zeros(M, N, device="cuda", dtype=torch.float32 if mode else torch.bfloat16)
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), G, M, N, K, d_rows=rows.data_ptr() if gather else 0, a_rows=a_rows, out_mode=mode)
    ctx.synchronize()
    p = picks(M)
    x = a[rows[p].long() if gather else p].double()
    for e, here in ((0, p < 200001), (2, p >= 200001)):
        check(out[p[here]], x[here] @ w[e].double().T, x[here].abs() @ w[e].double().abs().T, mode != 0)


def test_rows_of_a_long_operand(ctx):
    import scriptrs_b200 as sb

    rows, N, K = 540003, 64, 4096
    g = gen(2)
    a = torch.zeros(rows, K, device="cuda").bfloat16()
    p = picks(rows)
    a[p] = randn(g, p.numel(), K).bfloat16()
    w, off = randn(g, 1, N, K, std=K ** -0.5).bfloat16(), i32([0, p.numel()])
    idx, out = p.int(), torch.zeros(p.numel(), N, device="cuda")
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), 1, p.numel(), N, K, d_rows=idx.data_ptr(), a_rows=rows, out_mode=1)
    ctx.synchronize()
    check(out, a[p].double() @ w[0].double().T, a[p].double().abs() @ w[0].double().abs().T, True)


@pytest.mark.parametrize("M", [30, 300])
def test_long_weights(ctx, M):
    import scriptrs_b200 as sb

    G, N, K = 70, 4096, 8192
    g = gen(3)
    a, w = randn(g, M, K).bfloat16(), torch.empty(G, N, K, device="cuda", dtype=torch.bfloat16)
    for e in range(G):
        w[e] = randn(g, N, K, std=K ** -0.5)
    off = i32([M * e // G for e in range(G + 1)])
    out = torch.zeros(M, N, device="cuda")
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), G, M, N, K, out_mode=1)
    ctx.synchronize()
    cut = off.tolist()
    for e in (0, 31, 32, 63, 64, 68, 69):
        if cut[e] < cut[e + 1]:
            x = a[cut[e]:cut[e + 1]].double()
            check(out[cut[e]:cut[e + 1]], x @ w[e].double().T, x.abs() @ w[e].double().abs().T, True)


def test_adapters_of_a_long_result(ctx):
    import scriptrs_b200 as sb

    M, N, K, r, n = 540003, 4096, 64, 8, 3
    g = gen(4)
    a, w = randn(g, M, K).bfloat16(), randn(g, N, K, std=K ** -0.5).bfloat16()
    down, up = randn(g, n, r, K, std=K ** -0.5).bfloat16(), randn(g, n, N, r, std=r ** -0.5).bfloat16()
    who = (torch.arange(M, device="cuda") // 1000 % (n + 1) - 1).int()
    out = torch.zeros(M, N, device="cuda", dtype=torch.bfloat16)
    size = sb.adapter_gemm_workspace(M, r)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    sb.adapter_gemm(ctx, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), who.data_ptr(), out.data_ptr(), n, r, M, N, K, work.data_ptr(), size)
    ctx.synchronize()
    p = picks(M)
    x = a[p].double()
    y, s = x @ w.double().T, x.abs() @ w.double().abs().T
    for e in range(n):
        here = who[p] == e
        y[here] += (x[here] @ down[e].double().T) @ up[e].double().T
        s[here] += (x[here].abs() @ down[e].double().abs().T) @ up[e].double().abs().T
    check(out[p], y, s, False)


@pytest.mark.parametrize("k", [1, 2, 4])
def test_weighted_sum_of_long_rows(ctx, k):
    import scriptrs_b200 as sb

    rows, cols = 540003, 4096
    g = gen(5)
    y = torch.zeros(rows, cols, device="cuda", dtype=torch.bfloat16)
    p = picks(rows)
    y[p] = randn(g, p.numel(), cols).bfloat16()
    slots, w = torch.full((rows, k), -1, dtype=torch.int32, device="cuda"), randn(g, rows, k)
    for j in range(k):
        slots[p, j] = p.roll(7 * j + 1).int()
    out = torch.full((rows, cols), 3.0, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    sb.combine_rows(ctx, y.data_ptr(), slots.data_ptr(), w.data_ptr(), out.data_ptr(), rows, k, cols, rows)
    ctx.synchronize()
    terms = y[slots[p].long()].double() * w[p].double()[:, :, None]
    far = (out[p].double() - terms.sum(1)).abs()
    assert bool((far <= (k + 2) * 2.0 ** -24 * terms.abs().sum(1) + 2.0 ** -8 * terms.sum(1).abs() + 1e-30).all())
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    untouched[p] = False
    assert float(out[untouched][::997].abs().max()) == 0.0


def test_route_of_long_logits(ctx):
    import scriptrs_b200 as sb

    T, E, k = 2200003, 1024, 2
    x = torch.empty(T, E, device="cuda", dtype=torch.bfloat16).normal_(generator=gen(6))
    i = dict(dtype=torch.int32, device="cuda")
    experts, weights, offsets, order, slots = torch.empty(T, k, **i), torch.empty(T, k, device="cuda"), torch.empty(E + 1, **i), torch.empty(T * k, **i), torch.empty(T, k, **i)
    size = sb.route_topk_workspace(T, E, k)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    sb.route_topk(ctx, x.data_ptr(), experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(), order.data_ptr(), slots.data_ptr(), T, E, k, work.data_ptr(), size,
                  bf16=True)
    ctx.synchronize()
    p = picks(T)
    best = torch.sort(x[p].float(), dim=1, descending=True, stable=True)
    assert torch.equal(best.indices[:, :k].int(), experts[p])
    assert float((torch.softmax(best.values[:, :k].double(), 1) - weights[p]).abs().max()) < 2e-6
    flat = experts.reshape(-1).long()
    places = torch.sort(flat, stable=True).indices
    assert torch.equal(order.long(), places // k)
    assert torch.equal(offsets[1:].long(), torch.bincount(flat, minlength=E).cumsum(0))
    assert torch.equal(slots.reshape(-1)[places].long(), torch.arange(T * k, device="cuda"))
