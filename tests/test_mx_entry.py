"""What the C entry points of the microscaled operators refuse, on the host: an address that a kernel could
not use never reaches one."""
import pytest

P = 1 << 20  # an address; nothing is read there


@pytest.fixture
def call():
    from vorotracing_b200 import mx
    from vorotracing_b200._lib import lib

    def f(name, *args):
        status = mx._call(name)(*args)
        return status, lib().vt_last_error().decode()

    return f


@pytest.mark.parametrize("outs", [40, 300])
def test_workspace_alignment_of_the_gradients(call, outs):
    n = call("vt_mx8_linear_bwd_workspace_bytes", 4096, 64, outs, 0)[0]

    def bwd(workspace):
        return call("vt_mx8_linear_bwd", P, outs, P, 64, 2, 4096, 64, outs, P, P, 0, P, P, P, workspace, n, None, None)

    for at in (1, 8, 16, 48):
        status, text = bwd(P + at)
        assert status == 1 and "32-byte aligned" in text


def test_workspace_alignment_of_the_4_bit_product(call):
    n = call("vt_mx4_linear_workspace_bytes", 20000, 64, 300, 0)[0]
    assert n
    for at in (1, 8, 24):
        status, text = call("vt_mx4_linear", P, 64, 2, 20000, 64, 300, P, P, None, 0, P, P + at, n, None, None)
        assert status == 1 and "16-byte aligned" in text


@pytest.mark.parametrize("dtype,off", [(0, 1), (0, 2), (1, 1), (2, 1)])
def test_matrices_start_on_an_element(call, dtype, off):
    """An address between two elements would make every access misaligned."""
    n = 64
    wrong = [("vt_mx8_checkpoint", P + off, dtype, 8, n, n, 0, P, P, P, None), ("vt_mx8_checkpoint", P, dtype, 8, n, n, 0, P + off, P, P, None),
             ("vt_mx8_act_bwd", P + off, dtype, 8, n, n, P, P, 0, P, None), ("vt_mx8_act_bwd", P, dtype, 8, n, n, P, P, 0, P + off, None),
             ("vt_mx8_dequantize", P, P, 8, n, dtype, P + off, None), ("vt_mx4_quantize", P + off, dtype, 8, n, n, P, P, None),
             ("vt_mx4_dequantize", P, P, 8, n, dtype, P + off, None)]
    if dtype:
        for i in range(5):
            at = [P + off if i == j else P for j in range(5)]
            wrong.append(("vt_mx8_linear_bwd", at[0], 16, at[1], n, dtype, 8, n, 16, P, P, 0, *at[2:], P, 1 << 30, None, None))
        for i in range(3):
            at = [P + off if i == j else P for j in range(3)]
            wrong.append(("vt_mx4_linear", at[0], n, dtype, 8, n, 16, P, P, at[1], 0, at[2], P, 1 << 30, None, None))
    for args in wrong:
        status, text = call(*args)
        assert status == 1 and "does not start on an element" in text, args


def test_matrices_whose_blocks_no_count_holds(call):
    for rows, cols in (((1 << 40) + 1, 1), (1 << 40, 33), (1 << 36, 1 << 10), (1 << 39, 1 << 30)):
        for args in (("vt_mx8_checkpoint", P, 2, rows, cols, cols, 0, P, P, P, None), ("vt_mx8_act_bwd", P, 2, rows, cols, cols, P, P, 0, P, None),
                     ("vt_mx8_dequantize", P, P, rows, cols, 2, P, None), ("vt_mx4_quantize", P, 2, rows, cols, cols, P, P, None),
                     ("vt_mx4_dequantize", P, P, rows, cols, 2, P, None)):
            status, text = call(*args)
            assert status == 1 and "too many rows" in text, args
