"""Entry points of products whose weights a row chooses: refusals (the arguments are checked before the context, so no GPU is
needed), workspace sizes, and the tile rule over every form of a call."""
import ctypes as C
import itertools
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20  # an address on every boundary; nothing reads it


def lib():
    from scriptrs_b200 import _lib

    return _lib.lib()


def message():
    return lib().sb_last_error().decode()


GROUPED = dict(ctx=None, a=P, lda=64, a_rows=10, rows=None, w=P, bias=P, rs=None, cs=None, off=P, groups=3, out=P, ldo=32, M=10, N=32, K=64, fp8=0,
               act=1, mode=0, alpha=1.0)
ADAPTER = dict(ctx=None, a=P, lda=64, w=P, bias=None, down=P, up=P, scale=None, who=P, n=3, rank=16, out=P, ldo=32, M=10, N=32, K=64, act=0, mode=1,
               alpha=1.0, work=P, size=1 << 20)
ROUTE = dict(ctx=None, logits=P, bf16=0, ld=8, rows=10, experts=8, k=2, normalize=1, ids=P, weights=P, off=P, order=P, slots=P, work=P, size=1 << 20)
COMBINE = dict(ctx=None, y=P, y_f32=0, ldy=32, y_rows=20, slots=P, weights=None, out=P, ldo=32, rows=10, k=2, cols=32, mode=0, alpha=1.0)


def call(name, base, **change):
    args = dict(base, **change)
    return getattr(lib(), name)(*args.values())


@pytest.mark.parametrize("change", [dict(M=-1), dict(N=0), dict(K=0), dict(groups=0), dict(groups=-3), dict(M=2 ** 31), dict(N=2 ** 31), dict(K=2 ** 31),
                                    dict(M=2 ** 30, N=2 ** 20, ldo=2 ** 20), dict(groups=2 ** 27), dict(K=60, lda=64), dict(lda=56), dict(lda=68), dict(ldo=31), dict(act=3),
                                    dict(act=-1), dict(mode=3), dict(mode=-1), dict(a=None), dict(w=None), dict(out=None), dict(off=None), dict(a=P + 8),
                                    dict(w=P + 2), dict(out=P + 1), dict(mode=1, out=P + 2), dict(bias=P + 2), dict(off=P + 1), dict(rows=P + 2), dict(a_rows=9),
                                    dict(a_rows=0, rows=P), dict(a_rows=2 ** 31), dict(rs=P), dict(cs=P), dict(fp8=1, K=72, lda=80), dict(fp8=1, lda=72),
                                    dict(fp8=1, rs=P + 2), dict(fp8=1, cs=P + 1)], ids=str)
def test_grouped_refusals(change):
    assert call("sb_grouped_gemm", GROUPED, **change) == 11
    assert "ctx" not in message()


@pytest.mark.parametrize("change", [dict(n=0), dict(n=2 ** 27), dict(rank=0), dict(rank=12), dict(rank=136), dict(down=None), dict(up=None), dict(who=None),
                                    dict(down=P + 8), dict(up=P + 4), dict(work=P + 8), dict(scale=P + 2), dict(who=P + 1), dict(K=65, lda=72), dict(lda=63),
                                    dict(ldo=16), dict(act=4), dict(mode=5), dict(M=-5)], ids=str)
def test_adapter_refusals(change):
    assert call("sb_adapter_gemm", ADAPTER, **change) == 11
    assert "ctx" not in message()


@pytest.mark.parametrize("change", [dict(rows=-1), dict(experts=0), dict(experts=1025, ld=2000), dict(k=0), dict(k=9), dict(k=17, experts=32, ld=32), dict(ld=7),
                                    dict(rows=2 ** 30), dict(logits=None), dict(ids=None), dict(weights=None), dict(off=None), dict(order=None),
                                    dict(slots=None), dict(logits=P + 2), dict(bf16=1, logits=P + 1), dict(off=P + 2), dict(work=P + 4)], ids=str)
def test_route_refusals(change):
    assert call("sb_route_topk", ROUTE, **change) == 11
    assert "ctx" not in message()


@pytest.mark.parametrize("change", [dict(rows=-1), dict(k=0), dict(cols=0), dict(ldy=31), dict(ldo=31), dict(mode=3), dict(y=None), dict(slots=None),
                                    dict(out=None), dict(y=P + 1), dict(y_f32=1, y=P + 2), dict(mode=1, out=P + 2), dict(slots=P + 2), dict(y_rows=-1),
                                    dict(k=2 ** 31 - 1, rows=1), dict(cols=2 ** 31 - 1, ldy=2 ** 31, ldo=2 ** 31)], ids=str)
def test_combine_refusals(change):
    assert call("sb_combine_rows", COMBINE, **change) == 11
    assert "ctx" not in message()


@pytest.mark.parametrize("name,base", [("sb_grouped_gemm", GROUPED), ("sb_adapter_gemm", ADAPTER), ("sb_route_topk", ROUTE), ("sb_combine_rows", COMBINE)])
def test_good_arguments_reach_the_context(name, base):
    assert call(name, base) == 11
    assert message() == "ctx is null"


def test_workspaces():
    L = lib()
    need = L.sb_adapter_gemm_workspace(10, 16)
    assert need >= 10 * 16 * 4
    assert call("sb_adapter_gemm", ADAPTER, size=need - 1) == 12 and call("sb_adapter_gemm", ADAPTER, work=None) == 12
    assert call("sb_adapter_gemm", ADAPTER, size=need) == 11 and message() == "ctx is null"
    need = L.sb_route_topk_workspace(1000, 8, 2)
    assert call("sb_route_topk", ROUTE, rows=1000, size=need - 1) == 12
    assert call("sb_route_topk", ROUTE, rows=1000, size=need) == 11 and message() == "ctx is null"
    assert L.sb_adapter_gemm_workspace(0, 16) == L.sb_adapter_gemm_workspace(-1, 16) == L.sb_adapter_gemm_workspace(5, 129) == 0
    assert L.sb_route_topk_workspace(5, 1025, 2) == L.sb_route_topk_workspace(0, 8, 2) == L.sb_route_topk_workspace(5, 8, 0) == 0
    for m, r in itertools.product((1, 127, 128, 129, 52360), (8, 16, 128)):
        assert L.sb_adapter_gemm_workspace(m, r) == 4 * m * r


def test_the_python_functions_raise():
    import scriptrs_b200 as sb

    class NoContext:
        handle = C.c_void_p()

    with pytest.raises(sb.ScriptrsError) as e:
        sb.grouped_gemm(NoContext, P, P, P, P, 3, 10, 32, 60)
    assert e.value.status == 11
    with pytest.raises(sb.ScriptrsError) as e:
        sb.adapter_gemm(NoContext, P, P, P, P, P, P, 3, 16, 10, 32, 64, P, 5)
    assert e.value.status == 12
    with pytest.raises(sb.ScriptrsError):
        sb.route_topk(NoContext, P, P, P, P, P, P, 10, 8, 9, P, 1 << 20)
    with pytest.raises(sb.ScriptrsError):
        sb.combine_rows(NoContext, P, P, P, P, 10, 0, 32, 20)


def test_tile_rule(tmp_path):
    """Every form of a call gets one of the tiles that the kernel has."""
    src = tmp_path / "rule.cpp"
    src.write_text('#include "%s/scriptrs_b200/csrc/rows_tile.h"\n#include <cstdio>\n' % ROOT + r"""
int main() {
    long n = 0;
    for (long M : {1L, 2L, 24L, 127L, 128L, 129L, 1000L, 13160L, 52360L, 2000000L})
        for (int N = 1; N < 5000; N = N * 5 / 4 + 1)
            for (int G : {1, 2, 31, 32, 33, 1000, 60000})
                for (int f32 = 0; f32 < 4; ++f32)
                    for (int sms : {20, 132, 148}) {
                        const sb::RowsTileShape t = sb::rows_tile(M, N, G, (f32 & 1) != 0, f32 > 1, sms); const int bn = t.bn;
                        if (t.ctas == 2 ? (f32 == 3 || bn != 256) : !(bn == 32 || bn == 64 || bn == 128 || (bn == 256 && !(f32 & 1)))) { std::printf("bad %ld %d %d %d\n", M, N, G, bn); return 1; }
                        ++n;
                    }
    std::printf("%ld\n", n);
    return 0;
}
""")
    exe = tmp_path / "rule"
    subprocess.run(["g++", "-std=c++17", "-O1", "-o", str(exe), str(src)], check=True)
    assert int(subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout) > 1000
