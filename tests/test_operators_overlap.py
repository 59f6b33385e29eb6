"""Which bindings of the block norm and the 4-bit product share memory: exactly
those with a byte in common, single rows beside the columns of a wider buffer
among them (struct checks on the CPU, one such call on the GPU)."""
import ctypes

import numpy as np
import pytest

import test_gpu_block_norm as norm
from test_gpu_parity import Scope
from test_operators_abi_cpu import Fake, norm_args, q4_args

BASE = 0x100000


def status(abi, name, desc):
    return getattr(abi.load(), f"pk_{name}_validate")(ctypes.byref(desc))


def accepted(abi, first, row_bytes, **over):
    """Whether a single row of gates `first` bytes into the buffer of the output
    (8 rows of 64 f16, 256 bytes apart) is accepted."""
    desc = abi.block_norm_desc(**norm_args(
        output=Fake(BASE, 7 * 256 + 128), output_stride=128, input=Fake(0x800000, 1024), gate_rows=0,
        gate=Fake(BASE + first, row_bytes), **over))
    return status(abi, "block_norm", desc) == abi.OK


def test_a_gate_row_beside_the_outputs_columns(abi):
    """A row of 128 bytes in a buffer whose rows hold the output in their first
    128 of 256: free in the second half, wherever the row starts."""
    taken = np.zeros(4096, bool)
    for row in range(8):
        taken[1024 + row * 256:1024 + row * 256 + 128] = True
    for first in range(-300, 2300, 2):
        free = not taken[1024 + first:1024 + first + 128].any()
        assert accepted(abi, first, 128) == free, first
        # the gate's stride does not change where a single row lies
        assert accepted(abi, first, 128, gate_stride=100) == free, first


def test_parameters_between_the_rows(abi):
    """Norm parameters (256 bytes) in the second half of rows of 512."""
    for first, free in ((128, True), (256, True), (4, False), (124, False), (260, False), (384, False), (640, True)):
        desc = abi.block_norm_desc(**norm_args(output=Fake(BASE, 7 * 512 + 128), output_stride=256,
                                               input=Fake(0x800000, 1024), gamma=Fake(BASE + first, 256)))
        assert (status(abi, "block_norm", desc) == abi.OK) == free, first


def test_a_bias_between_the_rows_of_the_product(abi):
    """A bias of 160 bytes between outputs of 80 bytes in rows of 256."""
    for first, free in ((80, True), (96, True), (100, False), (76, False), (336, True), (7 * 256 + 80, True)):
        desc = abi.q4_desc(**q4_args(output=Fake(BASE, 7 * 256 + 80), output_stride=128, a=Fake(0x800000, 1024),
                                     bias=Fake(BASE + first, 160)))
        assert (status(abi, "q4", desc) == abi.OK) == free, first


@pytest.mark.gpu
def test_gate_row_and_outputs_in_one_buffer(abi, ctx):
    """One gate row for all rows, in the columns beside the output's."""
    case = norm.make(np.random.default_rng(1), np.float16, 9, 320, gate="all")
    scope = Scope(ctx)
    whole = np.full((9, 640), 77, np.float16)
    whole[4, 320:] = case["gate"][0]
    both = scope.put(whole)

    class View:
        dtype = np.dtype(np.float16)

        def __init__(self, at, nbytes):
            self.ptr, self.nbytes = both.ptr + at, nbytes
    nxt = scope.empty((9, 320), np.float16)
    put = {n: scope.put(case[n]) for n in ("input", "gamma", "beta", "residual", "next_gamma", "next_beta")}
    op = abi.BlockNormOp(ctx, rows=9, channels=320, gate=View(4 * 1280 + 640, 640), gate_rows=0, gate_stride=640,
                         output=View(0, 8 * 1280 + 640), output_stride=640, next_output=nxt, residual_scale=0.5, **put)
    op.enqueue()
    ctx.synchronize()
    op.release()
    got = both.download().reshape(9, 640)
    norm.check([got[:, :320], nxt.download()], case)
    assert (got[4, 320:] == case["gate"][0]).all() and (np.delete(got[:, 320:], 4, 0) == 77).all()
    scope.close()
