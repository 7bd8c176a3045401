#!/usr/bin/env python
"""Generates bindings/hearth-b200-sys/src/lib.rs, the Rust FFI declarations of every function, status code and
constant that include/hb200.h declares.

    python bindings/generate.py            # rewrite src/lib.rs
    python bindings/generate.py --check    # exit 1 if src/lib.rs is out of date

The crate is what a Hearth maintainer adds to the workspace next to hearth-quant / hearth-compute: a `-sys` crate
holding only `extern "C"` declarations, linked against libhearth_b200.so by its build.rs.  No Rust toolchain is
needed to generate it, and tests/test_bindings.py checks name and arity of every declaration against the header.
"""
from __future__ import annotations

import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(os.path.dirname(HERE), "include", "hb200.h")
OUT = os.path.join(HERE, "hearth-b200-sys", "src", "lib.rs")

SCALARS = {"int": "c_int", "size_t": "usize", "float": "f32", "double": "f64", "uint8_t": "u8", "int8_t": "i8",
           "uint32_t": "u32", "int32_t": "i32", "uint64_t": "u64", "char": "c_char", "void": "c_void"}
HANDLES = {"hb200_weight_t": "hb200_weight", "hb200_act_t": "hb200_act", "hb200_batch_t": "hb200_batch",
           "hb200_gguf_t": "hb200_gguf", "hb200_weight_i8_t": "hb200_weight_i8", "hb200_act_i8_t": "hb200_act_i8"}


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", "", text, flags=re.S)


def prototypes(text: str):
    """[(name, return type text, [argument text, ...])] in header order."""
    out = []
    body = re.sub(r"^\s*#.*$", "", strip_comments(text), flags=re.M)  # no preprocessor lines
    for m in re.finditer(r"HB200_API\s+([\w\s\*]+?)\b(hb200_\w+)\s*\((.*?)\)\s*;", body, flags=re.S):
        ret, name, args = m.group(1).strip(), m.group(2), " ".join(m.group(3).split())
        arglist = [] if args in ("", "void") else [a.strip() for a in args.split(",")]
        out.append((name, " ".join(ret.split()), arglist))
    return out


def rust_type(ctype: str) -> str:
    """C type text without the parameter name -> Rust type."""
    t = ctype.replace("*", " * ").split()
    # pointer levels read right to left: each '*' may be followed by 'const' (a const pointer, irrelevant to Rust)
    base, consts, stars = [], [], []
    i = 0
    while i < len(t) and t[i] != "*":
        (consts if t[i] == "const" else base).append(t[i])
        i += 1
    while i < len(t):
        if t[i] == "*":
            stars.append(False)
        elif t[i] == "const" and stars:
            stars[-1] = True
        i += 1
    b = " ".join(base)
    if b in HANDLES:
        r, base_const = f"*mut {HANDLES[b]}", False
    else:
        r, base_const = SCALARS[b], bool(consts)
    for k, _ in enumerate(stars):  # level k points at: the base (k == 0) or pointer level k - 1, either of them const or not
        pointee_const = base_const if k == 0 else stars[k - 1]
        r = f"*{'const' if pointee_const else 'mut'} {r}"
    return r


def split_arg(arg: str):
    """'const uint8_t handle[HB200_PEER_HANDLE_BYTES]' -> ('const uint8_t *', 'handle')."""
    m = re.match(r"^(.*?)(\w+)\s*(\[[^\]]*\])?$", arg)
    ctype, name, arr = m.group(1).strip(), m.group(2), m.group(3)
    if arr:
        ctype += " *"
    return ctype, name


def constants(text: str):
    text = strip_comments(text)
    status = re.search(r"typedef enum hb200_status \{(.*?)\}", text, flags=re.S).group(1)
    ids = re.search(r"\benum \{(.*?)\};", text, flags=re.S).group(1)
    items = [(k, int(v)) for k, v in re.findall(r"(HB200_\w+)\s*=\s*(-?\d+)", status + ids)]
    items += [(k, int(v)) for k, v in re.findall(r"#define\s+(HB200_\w+)\s+(\d+)\s*$", text, flags=re.M)]
    return items


def generate() -> str:
    text = open(HEADER).read()
    lines = [
        "//! Raw FFI declarations of libhearth_b200.so (include/hb200.h): the B200 implementation of Hearth's quantized",
        "//! matrix-product path.  Generated by bindings/generate.py from the header; do not edit by hand.",
        "#![allow(non_camel_case_types)]",
        "",
        "use core::ffi::{c_char, c_int, c_void};",
        "",
    ]
    for h in HANDLES.values():
        lines += ["#[repr(C)]", f"pub struct {h} {{", "    _private: [u8; 0],", "}"]
    lines.append("")
    for k, v in constants(text):
        ty = "usize" if k.startswith(("HB200_NOALLOC", "HB200_MAX", "HB200_PEER", "HB200_I8")) else "c_int"
        lines.append(f"pub const {k}: {ty} = {v};")
    lines += ["", '#[link(name = "hearth_b200")]', 'extern "C" {']
    for name, ret, args in prototypes(text):
        params = []
        for a in args:
            ctype, pname = split_arg(a)
            params.append(f"{pname}: {rust_type(ctype)}")
        r = "" if ret == "void" else f" -> {rust_type(ret)}"
        lines.append(f"    pub fn {name}({', '.join(params)}){r};")
    lines += ["}", ""]
    return "\n".join(lines)


if __name__ == "__main__":
    src = generate()
    if "--check" in sys.argv:
        sys.exit(0 if os.path.exists(OUT) and open(OUT).read() == src else 1)
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    open(OUT, "w").write(src)
    print(OUT)
