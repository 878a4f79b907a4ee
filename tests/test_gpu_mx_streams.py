"""Every kernel of the microscaled operators on a side stream, in a graph and from several threads: calls of more
than one launch over one workspace, and the ones before them whose results they read."""
import threading

import pytest
import torch

from test_gpu_mx import no_kernel_gave_up, values  # noqa: F401

pytestmark = pytest.mark.gpu

# (rows, cols, outs): few rows; one CTA a tile; with rows copied to whole words; pairs of CTAs and k split in the gradients
SHAPES = [(300, 128, 64), (9700, 96, 48), (9700, 91, 200), (5000, 96, 512), (3001, 48, 427), (5001, 300, 600), (20001, 24, 8)]


def operands(rows, cols, outs):
    return (values(rows, cols, torch.bfloat16, scale=1.0), values(rows, outs, torch.bfloat16, 1, 0.5), values(outs, cols, torch.bfloat16, 2, 0.3),
            values(1, outs, torch.bfloat16, 3)[0])


def step(z, dy, w, b):
    from vorotracing_b200 import mx

    h, ckpt = mx.act_checkpoint(z, "silu")
    w4 = mx.quantize4(w)
    return (h, mx.act_backward(z, ckpt), ckpt.dequantize(), *mx.linear_backward(dy, w, ckpt), w4.dequantize(), mx.linear4(z, w4, b, "silu"))


def equal(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("rows,cols,outs", SHAPES)
def test_side_stream(rows, cols, outs):
    args = operands(rows, cols, outs)
    want = step(*args)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        late = [torch.full_like(t, float("nan")) for t in args]
        torch.cuda._sleep(4_000_000)
        for a, b in zip(late, args):
            a.copy_(b)  # behind the sleep
        got = step(*late)
    torch.cuda.current_stream().wait_stream(s)
    equal(got, want)


@pytest.mark.parametrize("rows,cols,outs", SHAPES)
def test_graph(rows, cols, outs):
    args = operands(rows, cols, outs)
    mine = [torch.zeros_like(t) for t in args]
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = step(*mine)
    for k in range(3):  # other inputs each time
        for a, b in zip(mine, args):
            a.copy_(b.roll(k, 0))
        g.replay()
        equal(got, step(*mine))


def test_threads():
    """Threads that call the operators at once, each on a stream of its own and with other sizes."""
    args = [operands(*s) for s in SHAPES]
    want = [step(*a) for a in args]
    torch.cuda.synchronize()
    failed = []

    def work(i):
        try:
            s = torch.cuda.Stream()
            with torch.cuda.stream(s):
                for k in range(10):
                    at = (i + k) % len(SHAPES)
                    got = step(*args[at])
                    s.synchronize()
                    equal(got, want[at])
        except BaseException as e:
            failed.append((i, repr(e)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
