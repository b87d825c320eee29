"""The ctypes mirrors of the operators' argument structs have the header's layout (CPU only)."""
import ctypes
import os
import shutil
import subprocess

import pytest

from flare_b200 import _lib, _ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PAIRS = {"LookupArgs": "flare_lookup_args", "LookupGradArgs": "flare_lookup_grad_args", "RecurrenceArgs": "flare_recurrence_args",
         "ProductArgs": "flare_product_args"}
VALUES = {"FLARE_F32": 0, "FLARE_F16": 1, "FLARE_BF16": 2, "FLARE_MICRO": _ops.MICRO, "FLARE_I32": 0, "FLARE_I64": 1,
          "FLARE_RECURRENCE_SPAN": _lib.RECURRENCE_SPAN, "FLARE_PRODUCT_ROWS": _lib.PRODUCT_ROWS}


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs a C compiler")
def test_ctypes_structs_match_the_header(tmp_path):
    lines, expect = ["#include <stddef.h>", "#include <stdio.h>", '#include "flare_b200.h"', "int main(void) {"], []
    for py, c in PAIRS.items():
        cls = getattr(_lib, py)
        lines.append(f'    printf("%zu\\n", sizeof({c}));')
        expect.append((f"sizeof({c})", ctypes.sizeof(cls)))
        for name, _ in cls._fields_:
            lines.append(f'    printf("%zu\\n", offsetof({c}, {name}));')
            expect.append((f"{c}.{name}", getattr(cls, name).offset))
    for name, value in VALUES.items():
        lines.append(f'    printf("%d\\n", {name});')
        expect.append((name, value))
    src, exe = tmp_path / "probe.c", tmp_path / "probe"
    src.write_text("\n".join(lines + ["    return 0;", "}"]) + "\n")
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert [(w, v) for w, v in expect] == [(w, g) for (w, _), g in zip(expect, got)]


def test_packed_arguments_have_the_structs_layout():
    for pack, cls in ((_lib.PACK_LOOKUP, _lib.LookupArgs), (_lib.PACK_LOOKUP_GRAD, _lib.LookupGradArgs),
                      (_lib.PACK_RECURRENCE, _lib.RecurrenceArgs), (_lib.PACK_PRODUCT, _lib.ProductArgs)):
        n = len(cls._fields_)
        raw = pack.pack(*range(1, n + 1))
        a = cls.from_buffer_copy(raw.ljust(ctypes.sizeof(cls), b"\0"))
        got = [getattr(a, name) for name, _ in cls._fields_]
        assert got == list(range(1, n + 1)) and ctypes.sizeof(cls) - len(raw) < 8


def test_packed_arguments_are_as_long_as_the_structs():
    """The library may copy a whole struct, so its padding has to be there."""
    for pack, cls in ((_lib.PACK_LOOKUP, _lib.LookupArgs), (_lib.PACK_LOOKUP_GRAD, _lib.LookupGradArgs),
                      (_lib.PACK_RECURRENCE, _lib.RecurrenceArgs), (_lib.PACK_PRODUCT, _lib.ProductArgs)):
        assert pack.size == ctypes.sizeof(cls), cls.__name__
