"""The constants that the header defines, in its generated mirrors, against the values that a C compiler gives them."""
import os
import re
import subprocess

import pytest

from conftest import ROOT

HEADER = os.path.join(ROOT, "include", "qasr_hip.h")


def by_the_compiler(tmp_path):
    names = re.findall(r"^#define\s+(QASR_\w+)[ \t]+\S", open(HEADER).read(), re.M)
    src, exe = tmp_path / "c.c", tmp_path / "c"
    src.write_text('#include <stdio.h>\n#include "qasr_hip.h"\nint main(void) {\n'
                   + "".join(f'    printf("{n} %lld\\n", (long long)({n}));\n' for n in names) + "    return 0;\n}\n")
    subprocess.run(["gcc", "-std=c99", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    return {n: int(v) for n, v in (line.split() for line in out.splitlines())}


def test_the_embedded_constants_are_the_header_s(tmp_path):
    block = re.search(r"<!-- ffi:begin -->\n```rust\n(.*?)```\n<!-- ffi:end -->", open(os.path.join(ROOT, "INTEGRATION.md")).read(), re.S).group(1)
    got = {n: int(v) for n, v in re.findall(r"^pub const (\w+): c_int = (-?\d+);$", block, re.M)}
    want = by_the_compiler(tmp_path)
    assert len(want) >= 20 and got == want


def consts(text):
    from qwenasr_amd import ffi_rust
    return dict(ffi_rust.parse("#define QASR_GUARD_H\n" + text + "\n")[0])


def test_values_that_are_more_than_a_number():
    assert consts("#define QASR_A (1 << 18)\n#define QASR_B (-3)   /* minus three */\n#define QASR_C 0x40\n#define QASR_D (QASR_A + QASR_C * 2)\n"
                  "#define QASR_E (1u << 4)") == {"QASR_A": "262144", "QASR_B": "-3", "QASR_C": "64", "QASR_D": "262272", "QASR_E": "16"}


@pytest.mark.parametrize("value", ["sizeof(int)", "QASR_UNKNOWN", "1.5f", '"text"', "(1 <<", "1 / 2", "(1 << 31)", "017"])
def test_values_that_are_not_understood_are_refused(value):
    with pytest.raises(ValueError):
        consts(f"#define QASR_A {value}")
