"""The Go binding against the header it binds, as text: there is no Go toolchain here to compile it."""
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _read(*at):
    with open(os.path.join(ROOT, *at)) as f:
        return f.read()


GO, HEADER = _read("strix-halo-vulkan_amd", "go", "hip", "hip.go"), re.sub(r"/\*.*?\*/", "", _read("include", "shv_hip.h"), flags=re.S)
HELPERS = {"fp": {"float *"}, "ip": {"int32_t *"}, "vp": {"void *"}}


def _fields(name):
    """Field -> its C type ("float *", "int32_t", ..) of an argument block."""
    body = re.search(r"typedef struct \{([^{}]*)\} %s;" % name, HEADER).group(1)
    out = {}
    for line in filter(None, (x.strip() for x in body.split(";"))):
        typ, names = re.match(r"((?:const\s+)?\w+)\s+(.*)", line, re.S).groups()
        for n in names.split(","):
            n = n.strip()
            out[re.sub(r"[*\s]|\[.*", "", n)] = typ.replace("const ", "") + (" *" if n.startswith("*") else "")
    return out


BLOCKS = re.findall(r"var a C\.(shv_\w+_args)\n(.*?)\n}", GO, re.S)


def test_the_blocks_are_found():
    names = {n for n, _ in BLOCKS}
    assert {"shv_page_plan_args", "shv_attn_paged_args", "shv_logprobs_args", "shv_gemv_q4k_args", "shv_attn_decode_args", "shv_qsa_index_args", "shv_attn_tree_args"} <= names


@pytest.mark.parametrize("name,body", BLOCKS, ids=[n for n, _ in BLOCKS])
def test_what_a_constructor_sets_is_what_the_header_names(name, body):
    fields = _fields(name)
    for line in body.splitlines():
        m = re.match(r"\s*((?:a\.\w+(?:, )?)+) = (.*)", line)
        if not m:
            continue
        left = [x.strip()[2:].lstrip("_") for x in m.group(1).split(",")]
        right, depth, part = [], 0, ""
        for ch in m.group(2) + ",":
            if ch == "," and depth == 0:
                right.append(part.strip())
                part = ""
                continue
            depth += (ch in "([") - (ch in ")]")
            part += ch
        assert len(left) == len(right), line
        for f, value in zip(left, right):
            assert f in fields, (name, f)
            helper = re.match(r"(fp|ip|vp)\(", value)
            if helper:
                assert fields[f] in HELPERS[helper.group(1)], (name, f, fields[f], value)
            pointer = re.match(r"\(\*C\.(\w+)\)\(", value)
            if pointer:
                assert fields[f] == pointer.group(1) + " *", (name, f, fields[f], value)
            cast = re.match(r"C\.(int32_t|int64_t|uint32_t|float)\(", value)
            if cast:
                assert fields[f] == cast.group(1), (name, f, fields[f], value)


@pytest.mark.parametrize("name", ["shv_page_plan_args", "shv_attn_paged_args", "shv_logprobs_args"])
def test_every_field_of_the_paged_ops_is_set(name):
    body = dict(BLOCKS)[name]
    missing = [f for f in _fields(name) if f != "reserved" and not re.search(r"\ba\.%s\b" % f, body)]
    assert not missing


def test_ops_named_in_go_are_the_headers():
    assert set(re.findall(r"C\.(SHV_OP_\w+)", GO)) <= set(re.findall(r"\b(SHV_OP_\w+)", HEADER))
