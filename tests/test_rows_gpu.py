"""Products whose weights a row chooses, through the C ABI, against plain implementations in 64 bits.

Tolerances.  Products of bf16 or e4m3 values are exact in 32 bits.  One MMA adds 16 (32) of them to the running sum, each addend
cut off at 24 bits of the largest: at most 17 * 2^-23 (33 * 2^-23) of S, the sum of the absolute products; a 32-bit result
is collected every 256 (512) columns of K, that is after 16 MMAs, so its error is below 16 * 33 * 2^-23 S < 2^-13 S whatever K,
in practice far less: the norm is held to 1e-5 as for the shared product.  bf16 results add one rounding, 2^-8 of the value
(2^-8 / sqrt(3) in the norm at most, below 4e-3), and sum all of K without a collection: K / 16 * 17 * 2^-23 S < 2^-10 S at
K = 4096 in the worst case.  The first product of a low-rank addition enters a 32-bit result as three bf16 terms, 2^-24 of it; a
bf16 result as one, 2^-8 |low| |U| = 4 * 2^-10 |low| |U| (in the norm again 2^-8 / sqrt(3) of an addition that is no larger than
the result: together with the result's own rounding 3.2e-3).  SiLU passes errors on with a factor below 1.1 and adds a few
2^-22 of its own."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

SILU, RELU = 1, 2


def act64(y, act):
    if act == SILU:
        return y * torch.sigmoid(y)
    return torch.relu(y) if act == RELU else y


def check(out, ref, size, f32):
    """out against ref, both [M, N]; size: sums of absolute products."""
    got, ref = out.double(), ref.double()
    assert torch.isfinite(got).all()
    far = (got - ref).abs()
    bound = (2.0 ** -13 if f32 else 2.0 ** -10) * 1.1 * size + (2.0 ** -20 if f32 else 1.01 * 2.0 ** -8) * ref.abs() + 1e-30
    assert bool((far <= bound).all()), float((far - bound).max())
    if ref.numel() and float(ref.norm()) > 0:
        assert float((got - ref).norm() / ref.norm()) < (1e-5 if f32 else 4e-3)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, std=1.0):
    return torch.randn(*shape, device="cuda", generator=g) * std


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def offsets_of(sizes, start=0):
    return i32((start + np.concatenate([[0], np.cumsum(sizes)])).tolist())


# ------------------------------------------------------------------------------------------------------------- router
def route_ref(x, k, normalize):
    """Plain restatement in 64 bits; x [T, E] numpy float64."""
    T, E = x.shape
    z = np.where(np.isnan(x), -np.inf, x)
    z = np.where(z == np.inf, np.finfo(np.float32).max, z)
    ids = np.argsort(-z, axis=1, kind="stable")[:, :k]
    top = np.take_along_axis(z, ids, 1)
    m = z.max(1, keepdims=True)
    with np.errstate(invalid="ignore", over="ignore"):
        p = np.where(np.isneginf(z), 0.0, np.exp(z - m))
    chosen = np.take_along_axis(p, ids, 1)
    whole = (chosen if normalize else p).sum(1, keepdims=True)
    w = np.divide(chosen, whole, out=np.zeros_like(chosen), where=whole > 0)
    ids = np.where(np.isneginf(top), -1, ids)
    w = np.where(ids < 0, 0.0, w)
    flat = ids.reshape(-1)
    taken = np.flatnonzero(flat >= 0)
    placed = taken[np.argsort(flat[taken], kind="stable")]
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[taken], minlength=E))])
    order, slots = np.full(T * k, -1), np.full(T * k, -1)
    order[:placed.size] = placed // k
    slots[placed] = np.arange(placed.size)
    return ids, w, offsets, order, slots.reshape(T, k)


def run_route(ctx, x, k, normalize, ld=None):
    import scriptrs_b200 as sb

    T, E = x.shape
    out = dict(experts=torch.full((T, k), 77, dtype=torch.int32, device="cuda"), weights=torch.full((T, k), 7.0, device="cuda"),
               offsets=torch.full((E + 1,), 77, dtype=torch.int32, device="cuda"), order=torch.full((T * k,), 77, dtype=torch.int32, device="cuda"),
               slots=torch.full((T, k), 77, dtype=torch.int32, device="cuda"))
    size = sb.route_topk_workspace(T, E, k)
    work = torch.full((size + 16,), 0x5a, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    sb.route_topk(ctx, x.data_ptr(), out["experts"].data_ptr(), out["weights"].data_ptr(), out["offsets"].data_ptr(), out["order"].data_ptr(),
                  out["slots"].data_ptr(), T, E, k, work.data_ptr(), size, ld=ld or x.stride(0), bf16=x.dtype == torch.bfloat16, normalize=normalize)
    ctx.synchronize()
    assert bool((work[size:] == 0x5a).all())
    return out


def check_route(out, x, k, normalize):
    ids, w, offsets, order, slots = route_ref(x.double().cpu().numpy(), k, normalize)
    assert np.array_equal(out["experts"].cpu().numpy(), ids)
    assert np.array_equal(out["offsets"].cpu().numpy(), offsets)
    assert np.array_equal(out["order"].cpu().numpy(), order)
    assert np.array_equal(out["slots"].cpu().numpy(), slots)
    # sums of up to 1024 exponentials, each a few units of 2^-24
    assert np.abs(out["weights"].cpu().numpy() - w).max(initial=0.0) < 2e-6


@pytest.mark.parametrize("T,E,k,bf16,normalize", [(1, 1, 1, False, True), (1, 4, 2, False, True), (24, 32, 2, False, True), (127, 33, 3, True, False),
                                                  (128, 64, 4, True, True), (129, 65, 8, False, False), (1000, 128, 4, True, False),
                                                  (777, 300, 16, False, True), (90, 20, 16, True, False), (128, 1024, 16, False, True), (3000, 1000, 16, True, False),
                                                  (140001, 9, 2, True, True), (20000, 256, 3, False, False), (300, 1024, 5, True, False), (5000, 7, 7, False, False)])
def test_route(ctx, T, E, k, bf16, normalize):
    g = gen(T * 31 + E)
    x = randn(g, T, E, std=1.5).to(torch.bfloat16 if bf16 else torch.float32)
    check_route(run_route(ctx, x, k, normalize), x, k, normalize)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("normalize", [False, True])
def test_route_ties_masks_and_odd_values(ctx, bf16, normalize):
    dtype = torch.bfloat16 if bf16 else torch.float32
    inf, nan = float("inf"), float("nan")
    low = torch.finfo(dtype).min
    x = torch.randint(-2, 3, (200, 12), device="cuda", generator=gen(5)).to(dtype)  # many equal logits
    x[0] = -inf
    x[1] = nan
    x[2] = low
    x[3] = inf
    x[4] = -inf
    x[4, 7] = -3.0
    x[5, :6] = nan
    x[6] = 0.0
    x[6, 1::2] = -0.0  # equal to 0: the order is that of the indices
    x[7, 3] = inf
    x[8] = low
    x[8, 11] = -inf
    x[9, 4] = 80.0
    check_route(run_route(ctx, x, 4, normalize), x, 4, normalize)


def test_route_row_pitch_and_no_rows(ctx):
    import scriptrs_b200 as sb

    wide = randn(gen(9), 150, 40)
    x = wide[:, 3:36]
    check_route(run_route(ctx, x, 3, True), x, 3, True)
    offsets = torch.full((6,), 9, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    sb.route_topk(ctx, 0, 0, 0, offsets.data_ptr(), 0, 0, 0, 5, 2, 0, 0)
    ctx.synchronize()
    assert bool((offsets == 0).all())


# ---------------------------------------------------------------------------------------------------- grouped product
def grouped_case(ctx, sizes, N, K, *, gather=0, fp8=False, act=0, mode=0, bias=True, alpha=1.0, pad_a=0, pad_o=0, start=0, tail=0, shift=0, seed=1,
                 offsets=None):
    """Groups of `sizes` rows from row `start` on, `tail` rows behind them; gather: rows of A, picked by an index."""
    import scriptrs_b200 as sb

    g = gen(seed + 13 * N + K)
    G, M = len(sizes), start + int(sum(sizes)) + tail
    a_rows = gather or max(M, 1)
    a = randn(g, a_rows, K + pad_a)
    w = randn(g, G, N, K, std=K ** -0.5)
    rs = cs = None
    if fp8:
        rs, cs = a[:, :K].abs().amax(1) / 448.0, w.abs().amax(2) / 448.0
        a, w = (a / rs[:, None]).to(torch.float8_e4m3fn), (w / cs[:, :, None]).to(torch.float8_e4m3fn)
    else:
        a, w = a.bfloat16(), w.bfloat16()
    b = randn(g, G, N, std=0.3) if bias else None
    rows = torch.randint(0, a_rows, (max(M, 1),), device="cuda", generator=g).int() if gather else None
    if gather and M > 4:
        rows[1], rows[3] = -1, a_rows  # outside: rows of zeros
    off = offsets_of(sizes, start) if offsets is None else offsets
    dt = torch.bfloat16 if mode == 0 else torch.float32
    flat = torch.full(((M + 1) * (N + pad_o) + 64,), 3.0, device="cuda", dtype=dt)
    out = flat[shift:shift + (M + 1) * (N + pad_o)].view(M + 1, N + pad_o)
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), G, M, N, K, d_rows=rows.data_ptr() if gather else 0,
                    a_rows=a_rows, lda=K + pad_a, ldo=N + pad_o, d_bias=b.data_ptr() if bias else 0, act=act, out_mode=mode, alpha=alpha, fp8=fp8,
                    d_row_scale=rs.data_ptr() if fp8 else 0, d_col_scale=cs.data_ptr() if fp8 else 0)
    ctx.synchronize()
    # nothing outside the groups' rows and the N columns
    assert bool((flat[:shift] == 3.0).all()) and bool((flat[shift + (M + 1) * (N + pad_o):] == 3.0).all())
    assert bool((out[M:] == 3.0).all()) and bool((out[:, N:] == 3.0).all()) and bool((out[:start] == 3.0).all())
    assert bool((out[M - tail:] == 3.0).all())
    at = start
    for e, n in enumerate(sizes):
        if n:
            if gather:
                r = rows[at:at + n].long()
                x = a.float()[r.clamp(0, a_rows - 1)].double()[:, :K] * ((r >= 0) & (r < a_rows)).double()[:, None]
                s = rs[r.clamp(0, a_rows - 1)].double() if fp8 else None
            else:
                x = a[at:at + n, :K].double()
                s = rs[at:at + n].double() if fp8 else None
            we = w[e].double()
            y, size = x @ we.T, x.abs() @ we.abs().T
            if fp8:
                f = s[:, None] * cs[e].double()
                y, size = y * f, size * f
            if bias:
                y, size = y + b[e].double(), size + b[e].double().abs()
            if mode:
                ref = alpha * act64(y, act) + (3.0 if mode == 2 else 0.0)
                size = abs(alpha) * size + (3.0 if mode == 2 else 0.0)
            else:
                ref = act64(y, act)
            check(out[at:at + n, :N], ref, size, mode != 0)
        at += n
    return out[:M, :N].clone()


RAGGED = [[1], [128], [129], [0, 5, 0, 0, 130, 1], [3] * 40, [0] * 33 + [7] + [0] * 40, [300, 0, 1, 255, 256, 257], [2, 1, 0, 4, 1, 1, 3, 0],
          [0] * 130 + [140, 0, 3] + [1] * 127 + [0] * 500 + [60], [1, 0, 2] * 100]


@pytest.mark.parametrize("sizes", RAGGED, ids=lambda s: "_".join(map(str, s[:6])))
@pytest.mark.parametrize("gather", [0, 90])
@pytest.mark.parametrize("mode", [0, 1])
def test_grouped_ragged(ctx, sizes, gather, mode):
    grouped_case(ctx, sizes, 256, 128, gather=gather, mode=mode, act=SILU)


@pytest.mark.parametrize("N,K", [(1, 8), (8, 16), (30, 24), (33, 72), (64, 640), (127, 64), (1030, 640), (640, 1024), (257, 200), (1000, 4096)])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_grouped_odd_sizes(ctx, N, K, mode):
    grouped_case(ctx, [5, 0, 140, 17], N, K, mode=mode, act=[0, RELU, SILU][mode], alpha=0.5)
    grouped_case(ctx, [5, 0, 140, 17], N, K, gather=50, mode=mode, bias=False)


@pytest.mark.parametrize("gather", [0, 333])
@pytest.mark.parametrize("N,K,mode", [(256, 128, 0), (1030, 640, 1), (640, 272, 2), (128, 16, 0), (1024, 4096, 0)])
def test_grouped_e4m3(ctx, gather, N, K, mode):
    grouped_case(ctx, [0, 100, 1, 260, 39], N, K, gather=gather, fp8=True, mode=mode, act=SILU)


@pytest.mark.parametrize("gather", [0, 64])
@pytest.mark.parametrize("mode", [0, 1])
def test_grouped_strides_and_boundaries(ctx, gather, mode):
    """Row pitches beyond the width, results off the 16-byte boundary, rows before and behind the groups left as they are."""
    grouped_case(ctx, [70, 60], 200, 64, gather=gather, mode=mode, pad_a=24, pad_o=8, start=3, tail=5)
    grouped_case(ctx, [70, 60], 200, 64, gather=gather, mode=mode, pad_a=8, pad_o=3, start=1, tail=200, shift=1)
    grouped_case(ctx, [70, 60], 201, 64, gather=gather, mode=mode, pad_o=1, shift=3)


@pytest.mark.parametrize("N,pad", [(203, 5), (201, 7), (1030, 10), (2, 6)])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_columns_behind_the_last_are_left(ctx, N, pad, mode):
    """Rows on 16-byte boundaries whose last column lies inside 16 bytes: what stands behind it stays."""
    grouped_case(ctx, [70, 300, 60], N, 64, mode=mode, pad_o=pad)
    grouped_case(ctx, [70, 300, 60], N, 64, mode=mode, gather=90, pad_o=pad)
    grouped_case(ctx, [20, 0, 12], N, 64, mode=mode, gather=90, pad_o=pad)
    adapter_case(ctx, [i // 90 % 3 - 1 for i in range(400)], 2, 16, N, 64, mode=mode, pad_o=pad)
    adapter_case(ctx, [i % 3 - 1 for i in range(32)], 2, 16, N, 64, mode=mode, pad_o=pad)


@pytest.mark.parametrize("M,N,K,G", [(9000, 1024, 512, 3), (20011, 512, 256, 9), (4000, 2048, 1024, 1)])
@pytest.mark.parametrize("gather", [0, 777])
def test_grouped_large(ctx, M, N, K, G, gather):
    cuts = np.sort(np.random.RandomState(M).randint(0, M, G - 1))
    sizes = np.diff(np.concatenate([[0], cuts, [M]])).tolist()
    grouped_case(ctx, sizes, N, K, gather=gather, act=SILU)
    grouped_case(ctx, sizes, N, K, gather=gather, mode=1)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("mode", [1, 2])
@pytest.mark.parametrize("sizes,N,K", [([13160], 1024, 1024), ([6000, 0, 1, 255, 7000], 1000, 640), ([1, 13000, 300], 1030, 528), ([20000], 1024, 64)])
def test_grouped_large_in_32_bits(ctx, sizes, N, K, mode, fp8):
    """Enough rows for tiles of 256 x 256, which keep 128 sums a thread: one and several collections, groups that end inside a tile."""
    grouped_case(ctx, sizes, N, K, mode=mode, fp8=fp8, act=SILU, alpha=0.5, start=2, tail=9, pad_o=N % 4)


@pytest.mark.parametrize("fp8", [False, True])
def test_gathered_short_tiles_over_many_turns_of_the_ring(ctx, fp8):
    """Tiles with rows for some of the gathering warps only, K of many turns of the operand ring, several tiles per CTA."""
    r = np.random.RandomState(4)
    for sizes in (r.randint(1, 130, 60), [33] * 50, [1, 300, 2, 257, 40, 0, 129] * 6):
        grouped_case(ctx, list(map(int, sizes)), 2048, 4096, gather=500, fp8=fp8)
    grouped_case(ctx, [5000, 5100, 4099, 3, 2900], 2048, 2048, gather=900, fp8=fp8)
    grouped_case(ctx, [5000, 5100, 4099, 3, 2900], 2048, 2048, gather=900, fp8=fp8, mode=1)


def test_grouped_empty_calls(ctx):
    import scriptrs_b200 as sb

    grouped_case(ctx, [0, 0, 0], 64, 64, tail=40)
    sb.grouped_gemm(ctx, 0, 0, 0, 0, 4, 0, 64, 64)
    ctx.synchronize()


def test_grouped_offsets_are_clamped(ctx):
    """Offsets beyond M or below zero cost rows, not memory."""
    import scriptrs_b200 as sb

    M, N, K = 100, 64, 64
    g = gen(3)
    a, w = randn(g, M, K).bfloat16(), randn(g, 3, N, K).bfloat16()
    flat = torch.full((M + 300, N), 3.0, device="cuda")
    out = flat[100:100 + M]
    off = i32([-50, 40, 2000, 5000])
    torch.cuda.synchronize()
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), 3, M, N, K, out_mode=1)
    ctx.synchronize()
    assert bool((flat[:100] == 3.0).all()) and bool((flat[100 + M:] == 3.0).all())
    ref = torch.cat([a[:40].double() @ w[0].double().T, a[40:].double() @ w[1].double().T])
    assert float((out.double() - ref).norm() / ref.norm()) < 1e-5


@pytest.mark.parametrize("mode", [0, 1])
def test_grouped_a_row_does_not_depend_on_its_place(ctx, mode):
    """The same row in tiles of every width, alone, at other places and through an index: the same bits."""
    import scriptrs_b200 as sb

    N, K = 1024, 1024
    g = gen(8)
    a, w = randn(g, 3000, K).bfloat16(), randn(g, 2, N, K, std=K ** -0.5).bfloat16()

    def run(n0, n1, idx=None):
        M = n0 + n1
        out = torch.zeros(M, N, device="cuda", dtype=torch.float32 if mode else torch.bfloat16)
        off = i32([0, n0, M])
        torch.cuda.synchronize()
        sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), 2, M, N, K, d_rows=idx.data_ptr() if idx is not None else 0,
                        a_rows=3000, out_mode=mode)
        ctx.synchronize()
        return out

    whole = run(3000, 0)
    for n in (1, 7, 130, 700, 1500):
        assert torch.equal(run(n, 0), whole[:n]), n
    idx = torch.randperm(3000, device="cuda", generator=g)[:999].int()
    assert torch.equal(run(999, 0, idx), whole[idx.long()])
    other = run(0, 3000)
    got = run(444, 556, idx)
    assert torch.equal(got[:444], whole[idx[:444].long()]) and torch.equal(run(0, 999, idx), other[idx.long()])


def test_grouped_masked_rows_do_not_spread(ctx):
    """NaN and inf in rows that no group takes, and in another group's weights, stay where they are."""
    import scriptrs_b200 as sb

    N, K = 128, 64
    g = gen(4)
    a, w = randn(g, 64, K).bfloat16(), randn(g, 3, N, K).bfloat16()
    ref = a.double() @ w[1].double().T
    a[20:] = float("nan")
    w[0], w[2] = float("inf"), float("nan")
    off = i32([0, 0, 20, 20])
    for rows in (0, torch.arange(64, dtype=torch.int32, device="cuda")):
        out = torch.full((64, N), 3.0, device="cuda")
        torch.cuda.synchronize()
        sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), out.data_ptr(), off.data_ptr(), 3, 64, N, K, out_mode=1,
                        d_rows=rows.data_ptr() if torch.is_tensor(rows) else 0)
        ctx.synchronize()
        assert float((out[:20].double() - ref[:20]).norm() / ref[:20].norm()) < 1e-5
        assert bool((out[20:] == 3.0).all())


# ------------------------------------------------------------------------------------------------------------ combine
@pytest.mark.parametrize("rows,k,cols", [(1, 1, 1), (24, 2, 1024), (77, 3, 640), (130, 4, 1030), (1000, 8, 72), (5, 16, 33), (3000, 2, 1016)])
@pytest.mark.parametrize("pad", [3, 4, 8])
@pytest.mark.parametrize("y_f32", [False, True])
@pytest.mark.parametrize("mode", [0, 1, 2])
def test_combine(ctx, rows, k, cols, y_f32, mode, pad):
    import scriptrs_b200 as sb

    g = gen(rows + cols)
    y_rows = rows * k + 3
    y = randn(g, y_rows, cols + 8).to(torch.float32 if y_f32 else torch.bfloat16)
    w = randn(g, rows, k)
    slots = torch.randint(0, y_rows, (rows, k), device="cuda", generator=g).int()
    slots[torch.rand(rows, k, device="cuda", generator=g) < 0.1] = -1
    slots[0, 0] = y_rows
    if rows > 2:
        slots[2] = -1  # a row without results
    y[y_rows - 1] = float("nan")
    slots[slots == y_rows - 1] = 0
    out = torch.full((rows + 1, cols + pad), 3.0, device="cuda", dtype=torch.bfloat16 if mode == 0 else torch.float32)
    for weights in (w, None):
        out.fill_(3.0)
        torch.cuda.synchronize()
        sb.combine_rows(ctx, y.data_ptr(), slots.data_ptr(), weights.data_ptr() if weights is not None else 0, out.data_ptr(), rows, k, cols, y_rows,
                        ldy=cols + 8, ldo=cols + pad, y_f32=y_f32, out_mode=mode, alpha=0.5)
        ctx.synchronize()
        ok = (slots >= 0) & (slots < y_rows)
        f = (w if weights is not None else torch.ones_like(w)).double() * ok.double()
        picked = y[:, :cols].double()[(slots * ok).long()]
        terms = picked * f[:, :, None]
        ref = 0.5 * terms.sum(1) + (3.0 if mode == 2 else 0.0)
        size = 0.5 * terms.abs().sum(1) + (3.0 if mode == 2 else 0.0)
        # k + 2 roundings of 2^-24 of the sum of absolute terms, and the one to bf16
        far = (out[:rows, :cols].double() - ref).abs()
        assert bool((far <= (k + 2) * 2.0 ** -24 * size + (2.0 ** -8 * ref.abs() if mode == 0 else 0.0) + 1e-30).all())
        assert bool((out[rows:] == 3.0).all()) and bool((out[:, cols:] == 3.0).all())


# ----------------------------------------------------------------------------------------------------------- adapters
def adapter_case(ctx, who, n_adapters, rank, N, K, *, act=0, mode=0, bias=True, scale=True, alpha=1.0, pad_a=0, pad_o=0, shift=0, seed=1, poison=None):
    import scriptrs_b200 as sb

    g = gen(seed + 7 * N + K + rank)
    M = len(who)
    ids = i32(who)
    a = randn(g, max(M, 1), K + pad_a).bfloat16()
    w = randn(g, N, K, std=K ** -0.5).bfloat16()
    down = randn(g, n_adapters, rank, K, std=K ** -0.5).bfloat16()
    up = randn(g, n_adapters, N, rank, std=rank ** -0.5).bfloat16()
    sc = torch.rand(n_adapters, device="cuda", generator=g) + 0.5 if scale else None
    b = randn(g, N, std=0.3) if bias else None
    x = a[:, :K].double()
    y, size = x @ w.double().T, x.abs() @ w.double().abs().T
    for n in range(n_adapters):
        here = ids == n
        if n == poison:
            down[n], up[n] = float("nan"), float("inf")
            continue
        if bool(here.any()):
            s = float(sc[n]) if scale else 1.0
            low = x[here] @ down[n].double().T
            y[here] += s * (low @ up[n].double().T)
            if mode == 0:
                size[here] += 4 * s * (low.abs() @ up[n].double().abs().T)  # `low` in bf16
            size[here] += s * ((x[here].abs() @ down[n].double().abs().T) @ up[n].double().abs().T)
    if bias:
        y, size = y + b.double(), size + b.double().abs()
    ref = alpha * act64(y, act) + (3.0 if mode == 2 else 0.0) if mode else act64(y, act)
    size = abs(alpha) * size + (3.0 if mode == 2 else 0.0) if mode else size
    dt = torch.bfloat16 if mode == 0 else torch.float32
    flat = torch.full(((M + 1) * (N + pad_o) + 64,), 3.0, device="cuda", dtype=dt)
    out = flat[shift:shift + (M + 1) * (N + pad_o)].view(M + 1, N + pad_o)
    need = sb.adapter_gemm_workspace(M, rank)
    work = torch.full((need + 16,), 0xff, dtype=torch.uint8, device="cuda")  # NaN wherever it is read unwritten
    torch.cuda.synchronize()
    sb.adapter_gemm(ctx, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), ids.data_ptr(), out.data_ptr(), n_adapters, rank, M, N, K,
                    work.data_ptr(), need, lda=K + pad_a, ldo=N + pad_o, d_scale=sc.data_ptr() if scale else 0, d_bias=b.data_ptr() if bias else 0,
                    act=act, out_mode=mode, alpha=alpha)
    ctx.synchronize()
    assert bool((work[need:] == 0xff).all())
    assert bool((flat[:shift] == 3.0).all()) and bool((flat[shift + (M + 1) * (N + pad_o):] == 3.0).all())
    assert bool((out[M:] == 3.0).all()) and bool((out[:, N:] == 3.0).all())
    keep = ids != poison if poison is not None else torch.ones_like(ids, dtype=torch.bool)
    check(out[:M, :N][keep], ref[keep], size[keep], mode != 0)
    return out[:M, :N].clone()


def runs(*pairs):
    return [a for a, n in pairs for _ in range(n)]


WHO = {
    "one": [0],
    "none": [-1] * 5,
    "streams": [(5 * i) % 24 for i in range(24)],
    "all_different": [i % 131 for i in range(128)],
    "interleaved": [i % 3 - 1 for i in range(300)],
    "clips": runs((2, 188), (0, 126), (-1, 90), (7, 1), (3, 300), (2, 60)),
    "ids_outside": [5, 131, -7, 2 ** 31 - 1, -2 ** 31, 0, 130, 5] * 20,
    "last_row_of_a_tile": runs((1, 127), (2, 1), (1, 128), (3, 1)),
}


@pytest.mark.parametrize("name", sorted(WHO))
@pytest.mark.parametrize("rank,mode", [(8, 0), (16, 1), (64, 0)])
def test_adapters(ctx, name, rank, mode):
    adapter_case(ctx, WHO[name], 131, rank, 256, 128, act=SILU, mode=mode)


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 96, 104, 128])
@pytest.mark.parametrize("mode", [0, 2])
def test_adapter_ranks(ctx, rank, mode):
    adapter_case(ctx, runs((1, 100), (0, 30), (4, 100)), 5, rank, 200, 520, mode=mode, act=RELU, alpha=0.5)


@pytest.mark.parametrize("N,K", [(1, 8), (30, 24), (127, 64), (1030, 640), (640, 1024), (1000, 4096)])
@pytest.mark.parametrize("mode", [0, 1])
def test_adapter_odd_sizes_and_strides(ctx, N, K, mode):
    who = runs((1, 40), (-1, 3), (0, 150))
    adapter_case(ctx, who, 2, 16, N, K, mode=mode, pad_a=8, pad_o=5, shift=1)
    adapter_case(ctx, who, 2, 16, N, K, mode=mode, bias=False, scale=False)


@pytest.mark.parametrize("M,N,K,rank,n", [(13160, 1024, 1024, 16, 70), (20000, 2048, 512, 64, 8), (3000, 4096, 1024, 32, 300), (5000, 512, 1000, 128, 4),
                                            (300, 4096, 1024, 8, 3), (700, 1024, 1024, 16, 5)])
def test_adapters_large(ctx, M, N, K, rank, n):
    r = np.random.RandomState(M)
    cuts = np.sort(r.randint(0, M, 71))
    who = r.randint(-1, n, 72)[np.searchsorted(cuts, np.arange(M), side="right")].tolist()
    adapter_case(ctx, who, n, rank, N, K, act=SILU)
    adapter_case(ctx, who, n, rank, N, K, mode=1)


@pytest.mark.parametrize("M", [1, 7, 32, 33])
@pytest.mark.parametrize("rank,N,K,mode", [(8, 1030, 640, 0), (24, 4096, 1024, 1), (128, 30, 72, 2), (16, 45000, 64, 0), (64, 20000, 64, 1), (40, 127, 1000, 0),
                                           (16, 100000, 32, 0)])
def test_adapters_of_a_few_streams(ctx, M, rank, N, K, mode):
    """Up to 32 rows take another path; more than one tile per CTA in the wide ones."""
    who = [(7 * i) % 12 - 1 for i in range(M)]
    adapter_case(ctx, who, 11, rank, N, K, mode=mode, act=SILU, alpha=0.5)
    adapter_case(ctx, who, 11, rank, N, K, mode=mode, poison=6, pad_o=3, shift=1)


@pytest.mark.parametrize("mode", [0, 1])
def test_a_broken_adapter_stays_with_its_rows(ctx, mode):
    adapter_case(ctx, runs((0, 50), (1, 20), (2, 30), (-1, 28)) + [0, 1, 2] * 10, 3, 16, 256, 128, mode=mode, poison=1)


@pytest.mark.parametrize("mode", [0, 1])
def test_a_broken_adapter_among_many_rows(ctx, mode):
    """The same in products large enough for tiles of 256 rows, with up to a hundred adapters in one."""
    r = np.random.RandomState(3)
    who = np.repeat(r.randint(-1, 90, 700), r.randint(1, 35, 700))
    who[5000:5600] = r.randint(-1, 90, 600)
    adapter_case(ctx, who.tolist(), 90, 16, 1024, 64, mode=mode, poison=7)


@pytest.mark.parametrize("rank,mode", [(8, 1), (40, 2), (128, 1)])
def test_adapters_large_in_32_bits(ctx, rank, mode):
    """Tiles of 256 x 256 with several adapters each, one of them broken, and rows without any; off the 16-byte boundaries too."""
    r = np.random.RandomState(rank)
    who = np.repeat(r.randint(-1, 60, 500), r.randint(1, 60, 500))[:13100]
    who[4000:4300] = r.randint(-1, 60, 300)
    adapter_case(ctx, who.tolist(), 60, rank, 1024, 576, mode=mode, act=SILU, alpha=0.5, poison=7)
    adapter_case(ctx, who.tolist(), 60, rank, 1000, 520, mode=mode, pad_a=8, pad_o=3, shift=1)


def test_rows_without_an_adapter_equal_the_shared_product(ctx):
    """Bit for bit the grouped product of one group, beside rows that have one."""
    import scriptrs_b200 as sb

    M, N, K = 500, 512, 256
    g = gen(2)
    a, w = randn(g, M, K).bfloat16(), randn(g, N, K, std=K ** -0.5).bfloat16()
    down, up = randn(g, 2, 16, K).bfloat16(), randn(g, 2, N, 16).bfloat16()
    who = i32([[-1, 0, 1, -1][(i // 7) % 4] for i in range(M)])
    work = torch.empty(sb.adapter_gemm_workspace(M, 16), dtype=torch.uint8, device="cuda")
    x, y = (torch.empty(M, N, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    off = i32([0, M])
    torch.cuda.synchronize()
    sb.adapter_gemm(ctx, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), who.data_ptr(), x.data_ptr(), 2, 16, M, N, K, work.data_ptr(),
                    work.numel())
    sb.grouped_gemm(ctx, a.data_ptr(), w.data_ptr(), y.data_ptr(), off.data_ptr(), 1, M, N, K)
    ctx.synchronize()
    assert torch.equal(x[who < 0], y[who < 0]) and not torch.equal(x[who == 0], y[who == 0])


# ------------------------------------------------------------------------------------------------------------ together
def test_expert_module_eager_captured_and_on_another_stream(ctx):
    """Router, both products and the weighted sum, as an expert feed-forward module uses them: against 64 bits, then the same
    calls captured into a graph and replayed on new inputs, on a stream of the caller's."""
    import scriptrs_b200 as sb

    T, E, k, D, FF = 333, 8, 2, 256, 512
    g = gen(12)
    w1, w2 = randn(g, E, FF, D, std=D ** -0.5).bfloat16(), randn(g, E, D, FF, std=FF ** -0.5).bfloat16()
    b1, b2 = randn(g, E, FF, std=0.1), randn(g, E, D, std=0.1)
    x, logits = torch.empty(T, D, device="cuda", dtype=torch.bfloat16), torch.empty(T, E, device="cuda")
    i = dict(dtype=torch.int32, device="cuda")
    experts, weights = torch.empty(T, k, **i), torch.empty(T, k, device="cuda")
    offsets, order, slots = torch.empty(E + 1, **i), torch.empty(T * k, **i), torch.empty(T, k, **i)
    h, y = torch.empty(T * k, FF, device="cuda", dtype=torch.bfloat16), torch.empty(T * k, D, device="cuda", dtype=torch.bfloat16)
    res = torch.empty(T, D, device="cuda")
    size = sb.route_topk_workspace(T, E, k)
    work = torch.empty(size, dtype=torch.uint8, device="cuda")

    def fill(seed):
        g2 = gen(seed)
        x.copy_(randn(g2, T, D))
        logits.copy_(randn(g2, T, E))
        logits[5] = -float("inf")  # a padded frame: no expert
        res.copy_(randn(g2, T, D))

    def module():
        sb.route_topk(ctx, logits.data_ptr(), experts.data_ptr(), weights.data_ptr(), offsets.data_ptr(), order.data_ptr(), slots.data_ptr(), T, E, k,
                      work.data_ptr(), size)
        sb.grouped_gemm(ctx, x.data_ptr(), w1.data_ptr(), h.data_ptr(), offsets.data_ptr(), E, T * k, FF, D, d_rows=order.data_ptr(), a_rows=T,
                        d_bias=b1.data_ptr(), act=SILU)
        sb.grouped_gemm(ctx, h.data_ptr(), w2.data_ptr(), y.data_ptr(), offsets.data_ptr(), E, T * k, D, FF, d_bias=b2.data_ptr())
        sb.combine_rows(ctx, y.data_ptr(), slots.data_ptr(), weights.data_ptr(), res.data_ptr(), T, k, D, T * k, out_mode=2, alpha=0.5)

    def reference():
        p = torch.softmax(logits.double(), 1)
        top, ids = p.topk(k, dim=1)
        top = top / top.sum(1, keepdim=True)
        out = res.double().clone()
        for j in range(k):
            for e in range(E):
                here = (ids[:, j] == e) & torch.isfinite(logits[:, 0])
                hh = act64(x[here].double() @ w1[e].double().T + b1[e].double(), SILU)
                out[here] += 0.5 * top[here, j, None] * (hh @ w2[e].double().T + b2[e].double())
        return out

    def far(ref, start):
        # two roundings to bf16 (h, y) of the added part
        return float((res.double() - ref).norm() / (ref - start).norm())

    fill(1)
    ref, start = reference(), res.double().clone()
    torch.cuda.synchronize()
    module()
    ctx.synchronize()
    assert far(ref, start) < 8e-3
    assert torch.equal(res[5], start[5].float())
    stream = torch.cuda.Stream()
    ctx.set_stream(stream.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        fill(2)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            module()
        for seed in (3, 4):
            fill(seed)
            ref, start = reference(), res.double().clone()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert far(ref, start) < 8e-3
        fill(5)
        ref, start = reference(), res.double().clone()
        torch.cuda.synchronize()
        module()
        stream.synchronize()
        assert far(ref, start) < 8e-3
    finally:
        ctx.set_stream(0)


def test_two_adapter_graphs_with_workspaces_of_their_own_run_at_once(ctx):
    import scriptrs_b200 as sb

    M, N, K, r, n = 2000, 512, 512, 16, 9
    stream = torch.cuda.Stream()
    made = []
    for seed in (1, 2):
        g = gen(seed)
        a, w = randn(g, M, K).bfloat16(), randn(g, N, K, std=K ** -0.5).bfloat16()
        down, up = randn(g, n, r, K, std=K ** -0.5).bfloat16(), randn(g, n, N, r, std=0.3).bfloat16()
        who = torch.randint(-1, n, (M // 50,), device="cuda", generator=g).repeat_interleave(50).int()
        size = sb.adapter_gemm_workspace(M, r)
        work, out = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.zeros(M, N, device="cuda")
        ref = a.double() @ w.double().T
        for e in range(n):
            here = who == e
            ref[here] += (a[here].double() @ down[e].double().T) @ up[e].double().T
        ctx.set_stream(stream.cuda_stream)
        try:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph, stream=stream):
                sb.adapter_gemm(ctx, a.data_ptr(), w.data_ptr(), down.data_ptr(), up.data_ptr(), who.data_ptr(), out.data_ptr(), n, r, M, N, K,
                                work.data_ptr(), size, out_mode=1)
        finally:
            ctx.set_stream(0)
        made.append((graph, out, ref, (a, w, down, up, who, work)))
    streams = [torch.cuda.Stream() for _ in made]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (graph, *_rest) in zip(streams, made):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, out, ref, _keep in made:
        assert float((out.double() - ref).norm() / ref.norm()) < 1e-5
