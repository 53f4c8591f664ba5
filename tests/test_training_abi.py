"""The ctypes mirrors of the training-step structs against the C header: every
field's offset and every struct's size, from a C program compiled here with
gcc; enum values; and a C99 translation unit that calls each entry point."""

import ctypes
import os
import shutil
import subprocess

import pytest

from rollfast_b200 import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
STRUCTS = [("rf_saved_activation", _lib.RfSavedActivation), ("rf_norm_param", _lib.RfNormParam),
           ("rf_block_norm", _lib.RfBlockNorm), ("rf_rows", _lib.RfRows)]
ENUMS = {"RF_INT8": _lib.RF_INT8, "RF_E4M3": _lib.RF_E4M3, "RF_IN_OUT": _lib.RF_IN_OUT, "RF_OUT_IN": _lib.RF_OUT_IN,
         "RF_RMS_NORM": _lib.RF_RMS_NORM, "RF_LAYER_NORM": _lib.RF_LAYER_NORM,
         "RF_GATE_IDENTITY": _lib.RF_GATE_IDENTITY, "RF_GATE_SIGMOID": _lib.RF_GATE_SIGMOID,
         "RF_GATE_TANH": _lib.RF_GATE_TANH}


def _run(tmp_path, body, link=False):
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    src, exe = tmp_path / "t.c", tmp_path / "t"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include <string.h>\n#include "rollfast_b200.h"\n'
                   "int main(void) {\n" + body + "\n  return 0;\n}\n")
    cmd = [cc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)]
    if link:
        d = os.path.dirname(_lib.LIB_PATH)
        cmd += ["-L", d, "-lrollfast_b200", f"-Wl,-rpath,{d}"]
    subprocess.run(cmd, check=True)
    return subprocess.run([str(exe)], check=True, capture_output=True, text=True, timeout=120).stdout.split()


def test_ctypes_mirrors_match_the_header(tmp_path):
    want, lines = [], []
    for cname, cls in STRUCTS:
        lines.append(f'  printf("%zu\\n", sizeof({cname}));')
        want.append(ctypes.sizeof(cls))
        for field, _ in cls._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({cname}, {field}));')
            want.append(getattr(cls, field).offset)
    for name, value in ENUMS.items():
        lines.append(f'  printf("%d\\n", (int){name});')
        want.append(value)
    assert [int(x) for x in _run(tmp_path, "\n".join(lines))] == want


def test_c_caller(tmp_path):
    """What a C host gets without a GPU: plans, and refusals instead of aborts."""
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    out = _run(tmp_path, """
  size_t n = 0;
  rf_block_norm p;
  rf_saved_activation s;
  memset(&p, 0, sizeof p);
  memset(&s, 0, sizeof s);
  printf("%d\\n", rf_weight_gradient_workspace_size(4096, 768, 768, (void*)4096, 768, RF_BF16, &n) == RF_OK && n > 0);
  printf("%d\\n", rf_block_norm_workspace_size(&p, &n) == RF_EINVAL && strlen(rf_last_error()) > 0);
  p.rows = 512; p.features = 768; p.gate_rows = 1; p.scale = 1.0f;
  printf("%d\\n", rf_block_norm_workspace_size(&p, &n) == RF_OK && n == 0);
  p.pre_weight.value = (void*)4096; p.pre_weight.grad = (void*)8192;
  printf("%d\\n", rf_block_norm_workspace_size(&p, &n) == RF_OK && n > 0);
  printf("%d\\n", rf_save_activation(NULL, 0, RF_BF16, &s, 0, 0, NULL) == RF_EINVAL);
  printf("%d\\n", rf_load_activation(&s, NULL, 0, RF_BF16, NULL) == RF_EINVAL);
  printf("%d\\n", rf_swiglu_forward(NULL, 0, NULL, 0, NULL, 0, RF_BF16, 1, 8, NULL, NULL, NULL) == RF_EINVAL);
  printf("%d\\n", rf_swiglu_backward(NULL, 0, NULL, NULL, NULL, 0, NULL, 0, RF_BF16, NULL, NULL) == RF_EINVAL);
  printf("%d\\n", rf_weight_gradient(&s, NULL, 0, RF_BF16, 8, RF_IN_OUT, NULL, NULL, 0, RF_F32, NULL, 0, NULL) == RF_EINVAL);
  printf("%d\\n", rf_block_norm_forward(&p, NULL, NULL, NULL, NULL, NULL, NULL, NULL, NULL) == RF_EINVAL);
  printf("%d\\n", rf_block_norm_backward(&p, NULL, NULL, NULL, NULL, NULL, NULL, NULL, 0, NULL) == RF_EINVAL);
  printf("%d\\n", rf_kernel_launch_count() == 0);""", link=True)
    assert out == ["1"] * 12
