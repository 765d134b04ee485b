"""Every struct that the ctypes binding declares, and every constant that it restates, against the header: the lists are read from the
binding and the header, so a new one cannot be left out."""

import ctypes as C
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "lcmhip.h")


@pytest.fixture(scope="module")
def hip():
    from lcm import _hip
    return _hip


def _c_name(ct):
    return "lcmhip_" + re.sub(r"(?<=[a-z])(?=[A-Z])|(?<=[A-Z])(?=[A-Z][a-z])", "_", ct.__name__).lower()


def _structs(hip):
    return [x for x in vars(hip).values() if isinstance(x, type) and issubclass(x, C.Structure) and x is not C.Structure]


def _constants(hip):
    """LCMHIP_X for every integer X of the binding, LCMHIP_X_Y for every Y of a dictionary X, as far as the header has the name."""
    text = re.sub(r"/\*.*?\*/", " ", open(HEADER).read(), flags=re.S)
    names = set(re.findall(r"\bLCMHIP_\w+", text))
    found = {}
    for name, value in vars(hip).items():
        if isinstance(value, int) and not isinstance(value, bool):
            found["LCMHIP_" + name] = value
        elif isinstance(value, dict) and name.isupper():
            found.update({f"LCMHIP_{name}_{key.upper()}": x for key, x in value.items()})
    return {name: value for name, value in found.items() if name in names}


def _differences(tmp_path, structs, constants):
    lines = ['#include "lcmhip.h"', "#include <stdio.h>", "#include <stddef.h>", "int main(void) {"]
    for ct in structs:
        lines.append(f'    printf("{_c_name(ct)} %zu 0\\n", sizeof({_c_name(ct)}));')
        for field, _ in ct._fields_:
            lines.append(f'    printf("{_c_name(ct)}.{field} %zu %zu\\n", offsetof({_c_name(ct)}, {field}), sizeof((({_c_name(ct)}*)0)->{field}));')
    lines += [f'    printf("{name} %ld 0\\n", (long)({name}));' for name in constants] + ["    return 0;", "}"]
    src, exe = tmp_path / "layouts.c", tmp_path / "layouts"
    src.write_text("\n".join(lines) + "\n")
    subprocess.run(["gcc", "-std=c99", "-pedantic", "-Wall", "-Wextra", "-Werror", "-I", os.path.dirname(HEADER), str(src), "-o", str(exe)],
                   check=True, capture_output=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout
    seen = {name: (int(a), int(b)) for name, a, b in (line.split() for line in out.splitlines())}
    want = {name: (value, 0) for name, value in constants.items()}
    for ct in structs:
        want[_c_name(ct)] = (C.sizeof(ct), 0)
        for field, _ in ct._fields_:
            want[f"{_c_name(ct)}.{field}"] = (getattr(ct, field).offset, getattr(ct, field).size)
    return {name: (seen[name], value) for name, value in want.items() if seen[name] != value}


def test_every_struct_and_constant_of_the_binding(tmp_path, hip):
    structs, constants = _structs(hip), _constants(hip)
    names = {_c_name(ct) for ct in structs}
    assert {"lcmhip_kv_pages", "lcmhip_paged_batch", "lcmhip_shared_prefix", "lcmhip_head_norm", "lcmhip_rotary", "lcmhip_model_desc"} <= names
    assert {"LCMHIP_NORM_NONE", "LCMHIP_ROTARY_PAIRS", "LCMHIP_ROTARY_HALVES", "LCMHIP_NORM_RMS", "LCMHIP_ACT_RELU"} <= set(constants)
    assert _differences(tmp_path, structs, constants) == {}
    # the header's structs that a caller fills are all there
    text = re.sub(r"/\*.*?\*/", " ", open(HEADER).read(), flags=re.S)
    assert set(re.findall(r"\}\s*(lcmhip_\w+)\s*;", text)) == names


def test_a_reordered_field_is_seen(tmp_path, hip):
    fields = list(hip.PagedBatch._fields_)
    fields[0], fields[1] = fields[1], fields[0]
    fields[3], fields[4] = fields[4], fields[3]
    moved = type("PagedBatch", (C.Structure,), {"_fields_": fields})
    wrong = _differences(tmp_path, [moved], {"LCMHIP_NORM_NONE": 0})
    assert set(wrong) == {"LCMHIP_NORM_NONE"} | {f"lcmhip_paged_batch.{name}" for name in ("page_table", "seq_lens", "n_seqs", "max_pages")}
