"""The kernels of the row products are set up by the first call that needs them, not by every context; that call may be captured.  In
processes of their own, where nothing has been loaded before."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

START = """
import sys
sys.path.insert(0, %r)
import torch
import scriptrs_b200 as sb
T, E, k, D, FF, r = 333, 8, 2, 256, 512, 16
g = torch.Generator(device="cuda").manual_seed(1)
rn = lambda *s, std=1.0: torch.randn(*s, device="cuda", generator=g) * std
i = dict(dtype=torch.int32, device="cuda")
x, logits = rn(T, D).bfloat16(), rn(T, E)
w1, w2, wd = rn(E, FF, D, std=D ** -0.5).bfloat16(), rn(E, D, FF, std=FF ** -0.5).bfloat16(), rn(D, D, std=D ** -0.5).bfloat16()
down, up, who = rn(4, r, D, std=D ** -0.5).bfloat16(), rn(4, D, r, std=0.3).bfloat16(), (torch.arange(T, device="cuda") // 20 %% 5 - 1).int()
experts, weights, offsets, order, slots = torch.empty(T, k, **i), torch.empty(T, k, device="cuda"), torch.empty(E + 1, **i), torch.empty(T * k, **i), torch.empty(T, k, **i)
h, y, res = torch.empty(T * k, FF, device="cuda").bfloat16(), torch.empty(T * k, D, device="cuda").bfloat16(), torch.zeros(T, D, device="cuda")
out = torch.zeros(T, D, device="cuda")
size, need = sb.route_topk_workspace(T, E, k), sb.adapter_gemm_workspace(T, r)
work, work2 = torch.empty(size, dtype=torch.uint8, device="cuda"), torch.empty(need, dtype=torch.uint8, device="cuda")
p = lambda t: t.data_ptr()
def module(ctx):
    sb.route_topk(ctx, p(logits), p(experts), p(weights), p(offsets), p(order), p(slots), T, E, k, p(work), size)
    sb.grouped_gemm(ctx, p(x), p(w1), p(h), p(offsets), E, T * k, FF, D, d_rows=p(order), a_rows=T, act=1)
    sb.grouped_gemm(ctx, p(h), p(w2), p(y), p(offsets), E, T * k, D, FF)
    sb.combine_rows(ctx, p(y), p(slots), p(weights), p(res), T, k, D, T * k, out_mode=1)
    sb.adapter_gemm(ctx, p(x), p(wd), p(down), p(up), p(who), p(out), 4, r, T, D, D, p(work2), need, out_mode=1)
free = lambda: torch.cuda.mem_get_info()[0]
torch.cuda.synchronize()
""" % ROOT


def run(code):
    done = subprocess.run([sys.executable, "-c", START + code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout[-2000:] + done.stderr[-2000:]
    assert done.stdout.split()[-1] == "fine"


def test_a_context_alone_does_not_load_the_row_products():
    run("""
ctx = sb.Context(0)
before = free()
sb.grouped_gemm(ctx, p(x), p(w1), p(h), p(offsets.zero_()), E, T * k, FF, D, d_rows=p(order.zero_()), a_rows=T)
assert free() < before, "nothing was loaded by the first call"
ctx.synchronize()
print("fine")
""")


@pytest.mark.parametrize("mode", ["global", "thread_local", "relaxed"])
def test_the_first_calls_of_a_process_may_be_captured(mode):
    run("""
ctx = sb.Context(0)
stream = torch.cuda.Stream()
ctx.set_stream(stream.cuda_stream)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph, stream=stream, capture_error_mode=%r):
    module(ctx)
graph.replay()
torch.cuda.synchronize()
a, b, o = res.clone(), out.clone(), order.clone()
for t in (res, out, order, h, y):
    t.zero_()
torch.cuda.synchronize()
second = sb.Context(0)
module(second)
second.synchronize()
assert float(a.abs().max()) > 0 and float(b.abs().max()) > 0
assert torch.equal(a, res) and torch.equal(b, out) and torch.equal(o, order)
ref = x.double() @ wd.double().T
for e in range(4):
    ref[who == e] += (x[who == e].double() @ down[e].double().T) @ up[e].double().T
assert float((b.double() - ref).norm() / ref.norm()) < 1e-5
print("fine")
""" % mode)
