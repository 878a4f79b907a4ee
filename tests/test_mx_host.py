"""Host side of the microscaled operators: argument checks without a GPU."""
import os
import re

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_codes_match_the_header():
    from vorotracing_b200 import mx

    text = open(os.path.join(ROOT, "include", "vorotracing_b200.h")).read()
    defs = {k: int(v) for k, v in re.findall(r"#define (VT_[A-Z0-9_]+) (\d+)", text)}
    for name, code in mx.ACTS.items():
        assert defs["VT_ACT_" + name.upper()] == code
    for t, name in ((torch.float32, "F32"), (torch.float16, "F16"), (torch.bfloat16, "BF16")):
        assert defs["VT_" + name] == mx._DTYPES[t]


def test_argument_counts_match_the_header():
    from vorotracing_b200 import mx

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "vorotracing_b200.h")).read(), flags=re.S)
    for name, args in mx._ARGS.items():
        decl = re.search(r"\b" + name + r"\s*\(([^;]*)\);", text).group(1)
        assert len(decl.split(",")) == len(args), name


def test_host_tensors_are_refused():
    from vorotracing_b200 import mx

    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    for f in (mx.act_checkpoint, mx.quantize4):
        with pytest.raises(RuntimeError, match="CUDA device"):
            f(x)
    with pytest.raises(RuntimeError, match="CUDA device"):
        mx.MX4(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8), 64)
    with pytest.raises(RuntimeError, match="take codes"):
        mx.Checkpoint(torch.zeros((4, 64), dtype=torch.int8), torch.zeros((4, 3), dtype=torch.uint8), 64, "relu")
    with pytest.raises(RuntimeError, match="unknown activation"):
        mx.Checkpoint(torch.zeros((4, 64), dtype=torch.int8), torch.zeros((4, 2), dtype=torch.uint8), 64, "swish")


def test_workspace_sizes_cover_the_layout():
    from vorotracing_b200 import mx

    n = mx._call("vt_mx4_linear_workspace_bytes")
    assert n(1, 4096, 4096, 1) == 0
    for rows, cols in ((9999, 1), (12345, 1000), (1 << 20, 192)):
        blocks = -(-cols // 32)
        assert n(rows, cols, 300, 0) >= rows * blocks * 17
        assert n(rows, cols, 8, 0) == 0 and n(rows, cols, 8, 1) >= rows * cols * 2
    n = mx._call("vt_mx8_linear_bwd_workspace_bytes")
    for rows, cols, outs in ((1, 1, 1), (1000, 200, 77), (1000, 200, 777)):
        assert n(rows, cols, outs, 1) - n(rows, cols, outs, 0) >= (rows * outs * 2 if outs > 8 else 0)
        if outs > 256:
            assert n(rows, cols, outs, 2) - n(rows, cols, outs, 0) >= cols * outs * 2
