"""Shared arrays of the kernels that are read or written by vectors: an array's own alignment is its element's, so a wider access needs one that is asked for."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "zgml_b200", "csrc")
BYTES = {"int8_t": 1, "uint8_t": 1, "char": 1, "bool": 1, "bf16": 2, "half": 2, "__half": 2, "__nv_bfloat16": 2, "int16_t": 2, "uint16_t": 2, "int": 4, "int32_t": 4, "uint32_t": 4, "unsigned": 4, "float": 4,
         "float2": 8, "double": 8, "uint64_t": 8, "u64": 8, "int2": 8, "uint2": 8, "float4": 16, "int4": 16, "uint4": 16, "double2": 16, "ulonglong2": 16}
DECLARED = re.compile(r"(?<!extern )__shared__\s+((?:__align__|alignas)\((\d+)\)\s+)?([A-Za-z_0-9]+)\s+([^;]+);")
WIDE = re.compile(r"reinterpret_cast<\s*(?:const\s+)?([A-Za-z_0-9]+)\s*\*>\(\s*&?([A-Za-z_0-9]+)\b")


def misaligned(text):
    """(array, its alignment, bytes of the access) of each vector access to a static shared array that the array's declaration does not carry, within the array's function."""
    found = []
    for m in DECLARED.finditer(text):
        align = int(m[2] or BYTES.get(m[3], 16))
        end = text.find("\n}", m.end())
        for name in re.findall(r"([A-Za-z_0-9]+)\s*\[", re.sub(r"\[[^\]]*\]", "[", m[4])):
            for use in WIDE.finditer(text[m.end():end if end >= 0 else len(text)]):
                if use[2] == name and BYTES.get(use[1], 0) > align:
                    found.append((name, align, BYTES[use[1]]))
    return found


@pytest.mark.parametrize("path", sorted(os.path.basename(p) for p in glob.glob(os.path.join(CSRC, "*.cu*"))))
def test_vectors_of_shared_arrays(path):
    with open(os.path.join(CSRC, path)) as f:
        assert not misaligned(f.read())


def test_what_is_found():
    at = "void f() {\n    %s;\n    *reinterpret_cast<%s*>(rows[lane]) = x;\n}\n"
    assert misaligned(at % ("__shared__ int8_t rows[16][16]", "int4")) == [("rows", 1, 16)]
    assert misaligned(at % ("__shared__ float other[4], rows[8]", "float4")) == [("rows", 4, 16)]
    for fine in (("__shared__ alignas(16) int8_t rows[16][16]", "int4"), ("__shared__ __align__(8) float rows[8]", "float2"), ("__shared__ float4 rows[8]", "const float4"), ("__shared__ uint32_t rows[8]", "float")):
        assert not misaligned(at % fine)
