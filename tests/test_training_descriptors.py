"""Descriptors of the training operators: the C header, its ctypes mirror and the packed form lie alike."""
import ctypes
import os
import subprocess

from localfold_b200 import _native as nat, training

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MIRRORS = {"lf_float8_matrix": nat.Float8Matrix, "lf_float8_encode_desc": nat.Float8EncodeDesc, "lf_float8_decode_desc": nat.Float8DecodeDesc,
           "lf_layer_norm_desc": nat.LayerNormDesc, "lf_layer_norm_backward_desc": nat.LayerNormBackwardDesc,
           "lf_float8_linear_desc": nat.Float8LinearDesc, "lf_float8_weight_gradient_desc": nat.Float8WeightGradientDesc}
PACKED = {nat.Float8EncodeDesc: training._ENCODE, nat.Float8DecodeDesc: training._DECODE, nat.LayerNormDesc: training._LAYER_NORM,
          nat.LayerNormBackwardDesc: training._LAYER_NORM_BACKWARD, nat.Float8LinearDesc: training._LINEAR,
          nat.Float8WeightGradientDesc: training._WEIGHT_GRADIENT}


def test_mirrors_match_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "localfold_pairstack.h"', "int main(void) {"]
    for name, mirror in MIRRORS.items():
        lines.append(f'  printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'  printf("{name} {field} %zu\\n", offsetof({name}, {field}));' for field, _ in mirror._fields_]
    source, binary = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("\n".join(lines + ["  return 0;", "}"]))
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), "-o", str(binary), str(source)], check=True)
    out = subprocess.run([str(binary)], check=True, capture_output=True, text=True).stdout.splitlines()
    assert len(out) > 60
    for line in out:
        name, field, value = line.split()
        assert int(value) == (ctypes.sizeof(MIRRORS[name]) if field == "size" else getattr(MIRRORS[name], field).offset), line


def leaves(structure):
    for name, kind in structure._fields_:
        value = getattr(structure, name)
        if isinstance(value, ctypes.Structure):
            yield from leaves(value)
        else:
            yield 0 if value is None else value


def test_packed_forms_match_the_mirrors():
    """Distinct values, read back through the structure."""
    for mirror, packed in PACKED.items():
        count = len(list(leaves(mirror())))
        values = [3 * i + 1 for i in range(count)]
        data = packed.pack(*values)
        assert len(data) == ctypes.sizeof(mirror)
        assert list(leaves(mirror.from_buffer_copy(data))) == values


def test_sizes_match_the_library():
    lib = nat.load()
    for rows in (1, 127, 128, 129, 1000000):
        for channels in (1, 16, 17, 128, 511, 512, 513, 4096):
            assert training._sizes(rows, channels) == (lib.lf_float8_code_bytes(rows, channels), lib.lf_float8_exponent_bytes(rows, channels))
