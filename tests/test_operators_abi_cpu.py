"""Contracts of the block norm, the 4-bit product and the token scores without
a device: struct layouts, refusals with their messages, and the packed format."""
import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Fake:
    def __init__(self, ptr, nbytes, dtype=np.float16):
        self.ptr, self.nbytes, self.dtype = ptr, nbytes, np.dtype(dtype)


def test_struct_layouts_match_the_c_compiler(abi, tmp_path):
    structs = {"pk_block_norm_desc": abi.BlockNormDesc, "pk_q4_desc": abi.Q4Desc, "pk_score_desc": abi.ScoreDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "pk_block_norm.h"', '#include "pk_q4.h"',
             '#include "pk_score.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, field, value = line.split()
        cls = structs[cname]
        assert int(value) == (ctypes.sizeof(cls) if field == "sizeof" else getattr(cls, field).offset), (cname, field)


def refused(abi, name, desc, error, message):
    with pytest.raises(error, match=re.escape(message)) as caught:
        abi.check(getattr(abi.load(), f"pk_{name}_validate")(ctypes.byref(desc)))
    assert type(caught.value) is error


# ---------------------------------------------------------------- block norm


def norm_args(rows=8, channels=64, elem=2, **over):
    dtype, size = (np.float16, np.float32)[elem // 4], rows * channels * elem
    kw = dict(rows=rows, channels=channels, input=Fake(0x100000, size, dtype), gamma=Fake(0x10000, 4 * channels),
              beta=Fake(0x12000, 4 * channels), gate=Fake(0x200000, size, dtype), residual=Fake(0x300000, size, dtype),
              output=Fake(0x400000, size, dtype), next_gamma=Fake(0x14000, 4 * channels),
              next_beta=Fake(0x16000, 4 * channels), next_output=Fake(0x500000, size, dtype), label="layer.3")
    return dict(kw, **over)


def test_block_norm_accepts(abi):
    def ok(**over):
        desc = abi.block_norm_desc(**norm_args(**over))
        abi.check(abi.load().pk_block_norm_validate(ctypes.byref(desc)))
    ok()
    ok(elem=4)
    ok(gamma=None, beta=None, gate=None, residual=None, next_gamma=None, next_beta=None, next_output=None)
    ok(gate=Fake(0x200000, 64 * 2), gate_rows=0)
    ok(gate=Fake(0x200000, 64 * 2 * 2), gate_rows=5)
    ok(output=Fake(0x100000, 1024), next_output=Fake(0x300000, 1024))
    # an output beside the input in one buffer, and rows that fill their stride
    ok(input=Fake(0x100000, 8 * 256), input_stride=128, output=Fake(0x100080, 8 * 256), output_stride=128)
    ok(channels=16384, rows=1, gamma=None, beta=None, next_gamma=None, next_beta=None, next_output=None)


@pytest.mark.parametrize("over,error,message", [
    (dict(rows=0), "PaletteRangeError", "Invalid block norm shape for layer.3"),
    (dict(rows=4194304), "PaletteRangeError", "Invalid block norm shape for layer.3"),
    (dict(channels=16385), "PaletteRangeError", "Invalid block norm shape for layer.3"),
    (dict(epsilon=-1.0), "PaletteError", "layer.3 epsilon must be a finite number of at least 0"),
    (dict(epsilon=float("nan")), "PaletteError", "layer.3 epsilon must be a finite number of at least 0"),
    (dict(residual_scale=float("inf")), "PaletteError", "layer.3 residual scale must be finite"),
    (dict(input=Fake(None, 0)), "PaletteError", "layer.3 needs an input and an output"),
    (dict(gamma=None), "PaletteError", "layer.3 has a beta without its gamma"),
    (dict(next_output=None), "PaletteError", "layer.3 needs next gamma and next output together"),
    (dict(beta=Fake(0x12000, 128)), "PaletteError", "layer.3 beta must be float32 [64], 256 bytes"),
    (dict(gamma=Fake(0x10002, 256)), "PaletteError", "layer.3 gamma must be aligned to its elements"),
    (dict(input=Fake(0x100001, 1024)), "PaletteError", "layer.3 input must be aligned to its elements"),
    (dict(input=Fake(0x100000, 1022)), "PaletteRangeError", "layer.3 input needs 1024 bytes; arena slice has 1022"),
    (dict(gate=Fake(0x200000, 126), gate_rows=0), "PaletteRangeError", "layer.3 gate needs 128 bytes"),
    (dict(gate=Fake(0x200000, 128), gate_rows=7), "PaletteRangeError", "layer.3 gate needs 256 bytes"),
    (dict(residual_stride=63), "PaletteRangeError", "layer.3 residual stride must be at least the channels"),
    (dict(output_stride=65), "PaletteRangeError", "layer.3 output needs 1038 bytes; arena slice has 1024"),
    (dict(output=Fake(0x100080, 1024)), "PaletteError", "layer.3 outputs must be the input or the residual"),
    (dict(output=Fake(0x100000, 2048), output_stride=128), "PaletteError",
     "layer.3 outputs must be the input or the residual"),
    (dict(next_output=Fake(0x200000, 1024)), "PaletteError", "layer.3 outputs must not overlap the gate"),
    (dict(next_output=Fake(0x400000, 1024)), "PaletteError", "layer.3 output and next output must not overlap"),
    (dict(output=Fake(0x11ff0, 1024)), "PaletteError", "layer.3 outputs must not overlap the norms' parameters"),
    (dict(input=Fake(0x100000, 8 * 256), input_stride=128, output=Fake(0x10007e, 8 * 256), output_stride=128),
     "PaletteError", "layer.3 outputs must be the input or the residual"),
])
def test_block_norm_refusals(abi, over, error, message):
    refused(abi, "block_norm", abi.block_norm_desc(**{**norm_args(), **over}), getattr(abi, error), message)


def test_block_norm_struct_fields(abi):
    desc = abi.block_norm_desc(**norm_args())
    for field, value, message in (("struct_size", 8, "pk_block_norm_desc.struct_size mismatch"),
                                  ("precision", 7, "layer.3 has an unsupported precision 7"),
                                  ("kind", 2, "layer.3 has an unsupported norm kind 2")):
        before = getattr(desc, field)
        setattr(desc, field, value)
        refused(abi, "block_norm", desc, abi.PaletteError, message)
        setattr(desc, field, before)


# ------------------------------------------------------------------------ q4


def q4_args(rows=8, inner=64, columns=40, group_size=32, elem=2, **over):
    dtype = (np.float16, np.float32)[elem // 4]
    groups = -(-inner // (group_size or inner))
    kw = dict(rows=rows, inner=inner, columns=columns, group_size=group_size,
              a=Fake(0x100000, rows * inner * elem, dtype), packed=Fake(0x200000, (inner * columns + 7) // 8 * 4),
              scales=Fake(0x300000, groups * columns * elem), offsets=Fake(0x400000, groups * columns * elem),
              output=Fake(0x500000, rows * columns * elem, dtype), bias=Fake(0x600000, columns * 4),
              residual=Fake(0x700000, rows * columns * elem, dtype), residual_scale=0.5, label="head")
    return dict(kw, **over)


def test_q4_accepts(abi):
    def ok(**over):
        desc = abi.q4_desc(**q4_args(**over))
        abi.check(abi.load().pk_q4_validate(ctypes.byref(desc)))
    ok()
    ok(elem=4, inner=1000, columns=333, group_size=0)
    ok(offsets=None, bias=None, residual=None, residual_scale=None)
    ok(rows=1, inner=1, columns=1)
    ok(output=Fake(0x700000, 640))
    ok(activation="relu", group_size=1 << 20)


@pytest.mark.parametrize("over,error,message", [
    (dict(rows=0), "PaletteRangeError", "Invalid q4 shape [0, 64, 40] for head"),
    (dict(rows=1048561), "PaletteRangeError", "Invalid q4 shape"),
    (dict(inner=1 << 20, columns=1 << 20), "PaletteRangeError", "Invalid q4 shape"),
    (dict(a_stride=16777217), "PaletteRangeError", "head inner and a stride must be at most 16777216"),
    (dict(group_size=16), "PaletteRangeError", "head group size must be a power of two from 32 on, or 0"),
    (dict(group_size=96), "PaletteRangeError", "head group size must be a power of two from 32 on, or 0"),
    (dict(residual_scale=float("nan")), "PaletteError", "head residual scale must be finite"),
    (dict(residual=None), "PaletteError", "head has a residual scale without a residual"),
    (dict(scales=None), "PaletteError", "head needs a, packed, scales and output"),
    (dict(a_stride=63), "PaletteRangeError", "head a stride must be at least its columns"),
    (dict(output=Fake(0x500001, 640)), "PaletteError", "head output must be aligned to its elements"),
    (dict(a=Fake(0x100000, 1022)), "PaletteRangeError", "head a needs 1024 bytes; arena slice has 1022"),
    (dict(residual_stride=41), "PaletteRangeError", "head residual needs 654 bytes; arena slice has 640"),
    (dict(packed=Fake(0x200000, 1284)), "PaletteError", "head packed must be 1280 bytes of whole words"),
    (dict(scales=Fake(0x300000, 158)), "PaletteError", "head scales and offsets must be [2, 40], 160 bytes"),
    (dict(offsets=Fake(0x400000, 80)), "PaletteError", "head scales and offsets must be [2, 40], 160 bytes"),
    (dict(bias=Fake(0x600000, 80)), "PaletteError", "head bias must be float32 [40], 160 bytes"),
    (dict(output=Fake(0x100200, 640)), "PaletteError", "head output must not overlap a"),
    (dict(output=Fake(0x700010, 640)), "PaletteError", "head output must be the residual or not overlap it"),
    (dict(output=Fake(0x600000, 640)), "PaletteError", "head output must not overlap the bias"),
])
def test_q4_refusals(abi, over, error, message):
    refused(abi, "q4", abi.q4_desc(**{**q4_args(), **over}), getattr(abi, error), message)


def test_q4_struct_fields(abi):
    desc = abi.q4_desc(**q4_args())
    for field, value, message in (("struct_size", 8, "pk_q4_desc.struct_size mismatch"),
                                  ("precision", -1, "head has an unsupported precision -1"),
                                  ("activation", 3, "head has an unsupported activation 3")):
        before = getattr(desc, field)
        setattr(desc, field, value)
        refused(abi, "q4", desc, abi.PaletteError, message)
        setattr(desc, field, before)


def test_pack_q4_is_lsb_first(abi):
    codes = np.arange(20) % 16
    words = abi.pack_q4(codes.reshape(4, 5))
    assert [hex(w) for w in words] == ["0x76543210", "0xfedcba98", "0x3210"]


# --------------------------------------------------------------------- score


def score_args(rows=8, columns=1025, stride=1032, elem=2, k=4, **over):
    kw = dict(rows=rows, columns=columns, row_stride=stride, alternatives=k,
              logits=Fake(0x100000, ((rows - 1) * (stride or columns) + columns) * elem,
                          (np.float16, np.float32)[elem // 4]),
              tokens=Fake(0x200000, 4 * rows), log_probs=Fake(0x201000, 4 * rows), entropies=Fake(0x202000, 4 * rows),
              top_tokens=Fake(0x203000, 4 * rows * k) if k else None,
              top_log_probs=Fake(0x204000, 4 * rows * k) if k else None, label="confidence")
    return dict(kw, **over)


def test_q4_launch_limit(abi):
    """Row and column counts whose tiles no launch holds."""
    columns = (1 << 28) - 16
    kw = dict(a=Fake(1 << 50, 1 << 40), packed=Fake(1 << 51, columns * 4), scales=Fake(1 << 52, columns * 2),
              output=Fake(1 << 53, 1 << 50), inner=8, columns=columns, group_size=0, precision="f16", label="wide")
    abi.check(abi.load().pk_q4_validate(ctypes.byref(abi.q4_desc(rows=128, **kw))))
    refused(abi, "q4", abi.q4_desc(rows=129, **kw), abi.PaletteRangeError, "Invalid q4 shape [129, 8, ")


def test_score_accepts(abi):
    def ok(**over):
        desc = abi.score_desc(**score_args(**over))
        abi.check(abi.load().pk_score_validate(ctypes.byref(desc)))
    ok()
    ok(k=0)
    ok(k=32, columns=1, stride=0)
    ok(elem=4, tokens=None, log_probs=None, entropies=None)
    ok(k=0, tokens=None, log_probs=None, temperature=0.5)
    ok(columns=5, logits=Fake(0x100802, (7 * 1032 + 5) * 2))  # the duration columns of a head row


@pytest.mark.parametrize("over,error,message", [
    (dict(rows=0), "PaletteRangeError", "Invalid token score shape for confidence"),
    (dict(columns=0), "PaletteRangeError", "Invalid token score shape for confidence"),
    (dict(row_stride=1024), "PaletteRangeError", "confidence row stride must be at least the columns"),
    (dict(alternatives=33), "PaletteRangeError", "confidence alternatives must be in [0, 32]"),
    (dict(temperature=0.0), "PaletteRangeError", "confidence temperature must be in [2^-20, 2^20]"),
    (dict(temperature=float("nan")), "PaletteRangeError", "confidence temperature must be in [2^-20, 2^20]"),
    (dict(temperature=-1.0), "PaletteRangeError", "confidence temperature must be in [2^-20, 2^20]"),
    (dict(logits=Fake(None, 0)), "PaletteError", "confidence needs logits"),
    (dict(tokens=None), "PaletteError", "confidence needs tokens and log probs together"),
    (dict(top_tokens=None), "PaletteError", "confidence needs top tokens and top log probs with alternatives"),
    (dict(alternatives=0), "PaletteError", "confidence needs top tokens and top log probs with alternatives"),
    (dict(alternatives=0, top_tokens=None, top_log_probs=None, tokens=None, log_probs=None, entropies=None),
     "PaletteError", "confidence has no outputs"),
    (dict(logits=Fake(0x100001, 1 << 20)), "PaletteError", "confidence logits must be aligned to their elements"),
    (dict(logits=Fake(0x100000, 16496)), "PaletteRangeError", "confidence logits needs 16498 bytes"),
    (dict(entropies=Fake(0x202002, 32)), "PaletteError", "confidence entropies must be aligned to its elements"),
    (dict(top_tokens=Fake(0x203000, 124)), "PaletteRangeError", "confidence top tokens needs 128 bytes"),
    (dict(entropies=Fake(0x201010, 32)), "PaletteError", "confidence outputs must not overlap each other or the inputs"),
    (dict(log_probs=Fake(0x100800, 32)), "PaletteError", "confidence outputs must not overlap each other or the inputs"),
])
def test_score_refusals(abi, over, error, message):
    refused(abi, "score", abi.score_desc(**{**score_args(), **over}), getattr(abi, error), message)


def test_score_struct_fields(abi):
    desc = abi.score_desc(**score_args())
    for field, value, message in (("struct_size", 8, "pk_score_desc.struct_size mismatch"),
                                  ("precision", 2, "confidence has an unsupported precision 2")):
        before = getattr(desc, field)
        setattr(desc, field, value)
        refused(abi, "score", desc, abi.PaletteError, message)
        setattr(desc, field, before)


@pytest.mark.parametrize("name", ["block_norm", "q4", "score"])
def test_null_arguments(abi, name):
    lib = abi.load()
    assert getattr(lib, f"pk_{name}_validate")(None) == abi.INVALID_ARGUMENT
    assert getattr(lib, f"pk_{name}_enqueue")(None, 0, None) == abi.INVALID_ARGUMENT
    assert getattr(lib, f"pk_{name}_destroy")(None) == abi.OK
    assert getattr(lib, f"pk_{name}_release")(None) == abi.OK
