"""Objects of the microscaled operators on the host: whose memory a call is given."""
import copy
import io
import pickle

import pytest
import torch


def made(kind, rows=5, cols=70):
    """An object as the operators make them, one buffer of codes and exponents, on the host."""
    from vorotracing_b200 import mx

    q = getattr(mx, kind).__new__(getattr(mx, kind))
    if kind == "Checkpoint":
        q.act, q._act = "silu", mx.ACTS["silu"]
    q._new(torch.empty(0), rows, cols)
    q._buf.copy_(torch.arange(q._buf.numel(), dtype=torch.int64) % 251)
    return q


def saved(q):
    f = io.BytesIO()
    torch.save(q, f)
    f.seek(0)
    return torch.load(f, weights_only=False)


COPIES = {"copy": copy.copy, "deepcopy": copy.deepcopy, "pickle": lambda q: pickle.loads(pickle.dumps(q)), "save": saved}


@pytest.mark.parametrize("seen", [False, True])  # whether codes and exponents were looked at before
@pytest.mark.parametrize("how", COPIES)
@pytest.mark.parametrize("kind", ["Checkpoint", "MX4"])
def test_a_copy_gives_its_own_memory_to_the_kernels(kind, how, seen, monkeypatch):
    from vorotracing_b200 import mx

    calls = []
    monkeypatch.setattr(mx, "_launch", lambda name, index, *args: calls.append(args))
    q = made(kind)
    if seen:
        q.codes, q.exps
    c = COPIES[how](q)
    assert torch.equal(c.codes, q.codes) and torch.equal(c.exps, q.exps) and (c.rows, c.cols) == (q.rows, q.cols)
    assert how == "copy" or c.codes.data_ptr() != q.codes.data_ptr()
    for x in (q, c):
        x.dequantize()
        assert calls.pop()[:2] == (x.codes.data_ptr(), x.exps.data_ptr())
    if kind == "Checkpoint":
        assert c.act == q.act and c._act == q._act


def test_what_was_loaded_to_the_host_is_refused():
    with pytest.raises(RuntimeError, match="CUDA device"):
        made("MX4").dequantize()
