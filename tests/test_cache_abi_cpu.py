"""Contracts of the cache append, the cache attention and the draft verification
without a device: struct layouts and refusals with their messages."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

from test_operators_abi_cpu import Fake, refused

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_struct_layouts_match_the_c_compiler(abi, tmp_path):
    structs = {"pk_cache_append_desc": abi.CacheAppendDesc, "pk_cache_attention_desc": abi.CacheAttentionDesc,
               "pk_verify_desc": abi.VerifyDesc}
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "pk_cache.h"', '#include "pk_verify.h"',
             "int main(void) {"]
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


# 11 rows of 3 sequences; 4 query heads over 2 kv heads of 64; 10 pages of 16 tokens, 5 of a sequence
PAGE = 2 * 16 * 64


def cache_args(elem=2, **over):
    dtype = (np.float16, np.float32)[elem // 4]
    kw = dict(rows=11, sequences=3, heads=4, kv_heads=2, head_dim=64, queries=Fake(0x100000, 11 * 256 * elem, dtype),
              row_starts=Fake(0x10000, 16), lengths=Fake(0x11000, 12), page_table=Fake(0x12000, 60),
              pages_per_sequence=5, pages=10, page_size=16, key_cache=Fake(0x1000000, 10 * PAGE * elem, dtype),
              value_cache=Fake(0x2000000, 10 * PAGE * elem, dtype), label="step")
    return dict(kw, **over)


def append_args(elem=2, **over):
    dtype = (np.float16, np.float32)[elem // 4]
    kw = dict(cache_args(elem), keys=Fake(0x200000, 11 * 128 * elem, dtype),
              values=Fake(0x300000, 11 * 128 * elem, dtype), query_output=Fake(0x400000, 11 * 256 * elem, dtype),
              rotary_dim=64, frequencies=Fake(0x13000, 128), positions=Fake(0x14000, 44))
    return dict(kw, **over)


def attention_args(elem=2, **over):
    return dict(cache_args(elem), **{"output": Fake(0x400000, 11 * 256 * elem, (np.float16, np.float32)[elem // 4]), **over})


CACHE_REFUSALS = [
    (dict(rows=0), "PaletteRangeError", "Invalid cache rows [3 sequences, 0] for step"),
    (dict(rows=1048577), "PaletteRangeError", "Invalid cache rows [3 sequences, 1048577] for step"),
    (dict(sequences=0), "PaletteRangeError", "Invalid cache rows [0 sequences, 11] for step"),
    (dict(sequences=4097), "PaletteRangeError", "Invalid cache rows [4097 sequences, 11] for step"),
    (dict(kv_heads=0), "PaletteRangeError", "Invalid cache heads [4 over 0, 64] for step"),
    (dict(heads=1026), "PaletteRangeError", "Invalid cache heads [1026 over 2, 64] for step"),
    (dict(head_dim=60), "PaletteRangeError", "Invalid cache heads [4 over 2, 60] for step"),
    (dict(head_dim=264), "PaletteRangeError", "Invalid cache heads [4 over 2, 264] for step"),
    (dict(head_dim=0), "PaletteRangeError", "Invalid cache heads [4 over 2, 0] for step"),
    (dict(page_size=0), "PaletteRangeError", "Invalid cache pages [10 of 0, 5 of a sequence] for step"),
    (dict(page_size=65537), "PaletteRangeError", "Invalid cache pages [10 of 65537, 5 of a sequence] for step"),
    (dict(pages=0), "PaletteRangeError", "Invalid cache pages [0 of 16, 5 of a sequence] for step"),
    (dict(pages_per_sequence=1 << 28), "PaletteRangeError", "Invalid cache pages"),
    (dict(lengths=None), "PaletteError", "step needs row starts, lengths, a page table and caches"),
    (dict(value_cache=None), "PaletteError", "step needs row starts, lengths, a page table and caches"),
    (dict(page_stride=PAGE - 8), "PaletteRangeError", "step page stride must be a multiple of 8 of at least a page"),
    (dict(page_stride=PAGE + 4), "PaletteRangeError", "step page stride must be a multiple of 8 of at least a page"),
    (dict(page_stride=1 << 62), "PaletteRangeError", "step page stride must be a multiple of 8 of at least a page"),
    (dict(page_stride=1 << 33), "PaletteRangeError", "step caches must be within 68719476736 bytes"),
    (dict(row_starts=Fake(0x10000, 12)), "PaletteRangeError", "step row starts needs 16 bytes; arena slice has 12"),
    (dict(lengths=Fake(0x11000, 8)), "PaletteRangeError", "step lengths needs 12 bytes; arena slice has 8"),
    (dict(page_table=Fake(0x12002, 60)), "PaletteError", "step page table must be aligned to its elements"),
    (dict(page_table=Fake(0x12000, 56)), "PaletteRangeError", "step page table needs 60 bytes; arena slice has 56"),
    (dict(key_cache=Fake(0x1000008, 1 << 20)), "PaletteError", "step key cache must be aligned to 16 bytes"),
    (dict(value_cache=Fake(0x2000000, 40958)), "PaletteRangeError", "step value cache needs 40960 bytes"),
    (dict(page_stride=PAGE + 8), "PaletteRangeError", "step key cache needs 41104 bytes; arena slice has 40960"),
    (dict(query_stride=255), "PaletteRangeError", "step queries stride must be at least its columns"),
    (dict(query_stride=257), "PaletteRangeError", "step queries needs 5652 bytes; arena slice has 5632"),
    (dict(queries=Fake(0x100001, 1 << 20)), "PaletteError", "step queries must be aligned to its elements"),
]


def accepts(abi, name, desc):
    abi.check(getattr(abi.load(), f"pk_{name}_validate")(ctypes.byref(desc)))


def test_cache_append_accepts(abi):
    def ok(**over):
        accepts(abi, "cache_append", abi.cache_append_desc(**append_args(**over)))
    ok()
    ok(elem=4)
    ok(positions=None)
    ok(heads=0, queries=None, query_output=None)
    ok(rotary_dim=0, frequencies=None, positions=None)
    ok(rotary="neighbours", rotary_dim=2)
    ok(query_output=Fake(0x100000, 5632))                 # in place
    # the parts of one product, rotated in place
    row = dict(query_stride=512, key_stride=512, value_stride=512, query_output_stride=512)
    ok(queries=Fake(0x100000, 12288), keys=Fake(0x100200, 11776), values=Fake(0x100300, 11520),
       query_output=Fake(0x100000, 12288), **row)
    # keys and values in halves of each page
    ok(page_stride=2 * PAGE, key_cache=Fake(0x1000000, 20 * PAGE * 2), value_cache=Fake(0x1000000 + PAGE * 2, 19 * PAGE * 2))
    ok(heads=3, queries=Fake(0x100000, 1 << 16), query_output=Fake(0x400000, 1 << 16))
    ok(pages=1, page_stride=1 << 36)                      # one page: no stride counts


@pytest.mark.parametrize("over,error,message", CACHE_REFUSALS + [
    (dict(queries=None), "PaletteError", "step needs queries and a query output with heads, and only then"),
    (dict(heads=0), "PaletteError", "step needs queries and a query output with heads, and only then"),
    (dict(keys=Fake(None, 0)), "PaletteError", "step needs keys and values"),
    (dict(rotary_dim=66), "PaletteRangeError", "step rotary dim must be even and at most 64"),
    (dict(rotary_dim=31), "PaletteRangeError", "step rotary dim must be even and at most 64"),
    (dict(frequencies=None), "PaletteError", "step needs frequencies with a rotary dim, and only then"),
    (dict(rotary_dim=0, positions=None), "PaletteError", "step needs frequencies with a rotary dim, and only then"),
    (dict(rotary_dim=0, frequencies=None), "PaletteError", "step has positions without a rotary dim"),
    (dict(frequencies=Fake(0x13000, 124)), "PaletteRangeError", "step frequencies needs 128 bytes"),
    (dict(positions=Fake(0x14000, 40)), "PaletteRangeError", "step positions needs 44 bytes"),
    (dict(key_stride=127), "PaletteRangeError", "step keys stride must be at least its columns"),
    (dict(values=Fake(0x300000, 2814)), "PaletteRangeError", "step values needs 2816 bytes"),
    (dict(query_output=Fake(0x400000, 5630)), "PaletteRangeError", "step query output needs 5632 bytes"),
    (dict(query_output=Fake(0x100200, 5632)), "PaletteError", "step query output must be the queries or not overlap them"),
    (dict(query_output=Fake(0x200000, 5632)), "PaletteError", "step query output must not overlap keys"),
    (dict(query_output=Fake(0x1000000, 5632)), "PaletteError", "step key cache must not overlap query output"),
    (dict(value_cache=Fake(0x1000000 + 4096, 40960)), "PaletteError", "step value cache must not overlap key cache"),
    (dict(keys=Fake(0x2000000, 2816)), "PaletteError", "step value cache must not overlap keys"),
    (dict(lengths=Fake(0x1000000, 12)), "PaletteError", "step key cache must not overlap lengths"),
])
def test_cache_append_refusals(abi, over, error, message):
    refused(abi, "cache_append", abi.cache_append_desc(**{**append_args(), **over}), getattr(abi, error), message)


def test_cache_attention_accepts(abi):
    def ok(**over):
        accepts(abi, "cache_attention", abi.cache_attention_desc(**attention_args(**over)))
    ok()
    ok(elem=4)
    ok(causal=False, score_cap=30.0, scale=-0.5)
    ok(window=1, scale=0.0)
    ok(query_stride=300, queries=Fake(0x100000, (10 * 300 + 256) * 2))
    ok(page_size=3, key_cache=Fake(0x1000000, 10 * 2 * 3 * 64 * 2), value_cache=Fake(0x2000000, 10 * 2 * 3 * 64 * 2))
    # queries and outputs as parts of one buffer's rows
    ok(query_stride=512, queries=Fake(0x100000, 12288), output=Fake(0x100200, 11776), output_stride=512)


@pytest.mark.parametrize("over,error,message", CACHE_REFUSALS + [
    (dict(heads=0), "PaletteRangeError", "step heads must be a multiple of the 2 kv heads"),
    (dict(heads=3), "PaletteRangeError", "step heads must be a multiple of the 2 kv heads"),
    (dict(rows=1 << 20, heads=64), "PaletteRangeError", "step has more than 4000000 blocks of 16 rows"),
    (dict(queries=Fake(None, 0)), "PaletteError", "step needs queries and an output"),
    (dict(window=5, causal=False), "PaletteError", "step has a window without causal"),
    (dict(scale=float("-inf")), "PaletteRangeError", "step scale must be at most 2^60 in magnitude"),
    (dict(scale=float("nan")), "PaletteRangeError", "step scale must be at most 2^60 in magnitude"),
    (dict(score_cap=-1.0), "PaletteRangeError", "step score cap must be 0 or in [2^-20, 2^20]"),
    (dict(score_cap=float("nan")), "PaletteRangeError", "step score cap must be 0 or in [2^-20, 2^20]"),
    (dict(output=Fake(0x400000, 5630)), "PaletteRangeError", "step output needs 5632 bytes"),
    (dict(output_stride=128), "PaletteRangeError", "step output stride must be at least its columns"),
    (dict(output=Fake(0x100000, 5632)), "PaletteError", "step output must not overlap queries"),
    (dict(output=Fake(0x2000000, 5632)), "PaletteError", "step output must not overlap value cache"),
    (dict(output=Fake(0x11000 - 5630, 5632)), "PaletteError", "step output must not overlap row starts"),
])
def test_cache_attention_refusals(abi, over, error, message):
    refused(abi, "cache_attention", abi.cache_attention_desc(**{**attention_args(), **over}), getattr(abi, error), message)


def verify_args(elem=2, **over):
    dtype = (np.float16, np.float32)[elem // 4]
    kw = dict(rows=12, sequences=3, columns=100, target=Fake(0x100000, 1200 * elem, dtype),
              draft=Fake(0x200000, 1200 * elem, dtype), row_starts=Fake(0x10000, 16), tokens=Fake(0x11000, 48),
              uniforms=Fake(0x12000, 48), draws=Fake(0x13000, 12), accepted=Fake(0x14000, 12),
              next_tokens=Fake(0x15000, 12), label="check")
    return dict(kw, **over)


def test_verify_accepts(abi):
    def ok(**over):
        accepts(abi, "verify", abi.verify_desc(**verify_args(**over)))
    ok()
    ok(elem=4, draft=None)
    ok(mode="greedy", draft=None, uniforms=None, draws=None)
    ok(mode="greedy")
    ok(temperature=2.0 ** -20)
    ok(target=Fake(0x100002, (11 * 208 + 100) * 2), target_stride=208)
    ok(columns=1, sequences=1)


@pytest.mark.parametrize("over,error,message", [
    (dict(rows=0), "PaletteRangeError", "Invalid draft verification shape [3 sequences, 0, 100] for check"),
    (dict(sequences=65536), "PaletteRangeError", "Invalid draft verification shape [65536 sequences, 12, 100] for check"),
    (dict(columns=0), "PaletteRangeError", "Invalid draft verification shape"),
    (dict(columns=16777217), "PaletteRangeError", "Invalid draft verification shape"),
    (dict(temperature=0.0), "PaletteRangeError", "check temperature must be in [2^-20, 2^20]"),
    (dict(temperature=float("nan")), "PaletteRangeError", "check temperature must be in [2^-20, 2^20]"),
    (dict(tokens=None), "PaletteError", "check needs target logits, row starts, tokens and outputs"),
    (dict(uniforms=None), "PaletteError", "check needs uniforms and draws"),
    (dict(target_stride=99), "PaletteRangeError", "check target stride must be at least the columns"),
    (dict(draft=Fake(0x200001, 4000)), "PaletteError", "check draft must be aligned to its elements"),
    (dict(draft_stride=101), "PaletteRangeError", "check draft needs 2422 bytes; arena slice has 2400"),
    (dict(row_starts=Fake(0x10000, 12)), "PaletteRangeError", "check row starts needs 16 bytes"),
    (dict(draws=Fake(0x13000, 8)), "PaletteRangeError", "check draws needs 12 bytes"),
    (dict(next_tokens=Fake(0x14008, 12)), "PaletteError", "check outputs must not overlap each other or the inputs"),
    (dict(accepted=Fake(0x100004, 12)), "PaletteError", "check outputs must not overlap each other or the inputs"),
])
def test_verify_refusals(abi, over, error, message):
    refused(abi, "verify", abi.verify_desc(**{**verify_args(), **over}), getattr(abi, error), message)


@pytest.mark.parametrize("name,desc,fields", [
    ("cache_append", lambda abi: abi.cache_append_desc(**append_args()),
     [("struct_size", 8, "pk_cache_append_desc.struct_size mismatch"), ("precision", 7, "step has an unsupported precision 7"),
      ("rotary", 2, "step has an unsupported rotary kind 2")]),
    ("cache_attention", lambda abi: abi.cache_attention_desc(**attention_args()),
     [("struct_size", 8, "pk_cache_attention_desc.struct_size mismatch"),
      ("precision", -1, "step has an unsupported precision -1"), ("causal", 2, "step causal must be 0 or 1")]),
    ("verify", lambda abi: abi.verify_desc(**verify_args()),
     [("struct_size", 8, "pk_verify_desc.struct_size mismatch"), ("precision", 2, "check has an unsupported precision 2"),
      ("mode", 2, "check has an unsupported mode 2")]),
])
def test_struct_fields(abi, name, desc, fields):
    for field, value, message in fields:
        d = desc(abi)
        setattr(d, field, value)
        refused(abi, name, d, abi.PaletteError, message)


@pytest.mark.parametrize("name", ["cache_append", "cache_attention", "verify"])
def test_null_arguments(abi, name):
    lib = abi.load()
    assert getattr(lib, f"pk_{name}_validate")(None) == abi.INVALID_ARGUMENT
    assert getattr(lib, f"pk_{name}_enqueue")(None, 0, None) == abi.INVALID_ARGUMENT
    assert getattr(lib, f"pk_{name}_destroy")(None) == abi.OK
    assert getattr(lib, f"pk_{name}_release")(None) == abi.OK
