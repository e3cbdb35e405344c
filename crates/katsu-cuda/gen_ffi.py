#!/usr/bin/env python3
"""Writes crates/katsu-cuda/src/ffi.rs, the `extern "C"` block of the katsu-cuda crate, from
include/katsu_cuda.h, so that the Rust declarations cannot drift from the C ABI.

    python crates/katsu-cuda/gen_ffi.py            rewrite src/ffi.rs
    python crates/katsu-cuda/gen_ffi.py --check    exit 1 if src/ffi.rs is out of date
"""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
HEADER = os.path.join(ROOT, "include", "katsu_cuda.h")
OUT = os.path.join(HERE, "src", "ffi.rs")

TYPES = {
    "int32_t": "i32", "uint64_t": "u64", "size_t": "usize", "float": "f32",
    "int32_t *": "*mut i32", "uint64_t *": "*mut u64", "float *": "*mut f32", "const float *": "*const f32",
    "float **": "*mut *mut f32", "void **": "*mut *mut c_void", "size_t *": "*mut usize",
    "int8_t *": "*mut i8", "const int8_t *": "*const i8", "const size_t *": "*const usize",
    "const int32_t *": "*const i32", "const uint32_t *": "*const u32",
    "float *const *": "*const *mut f32", "const float *const *": "*const *const f32",
    "katsu_cuda_ctx *": "*mut Ctx", "katsu_cuda_ctx **": "*mut *mut Ctx",
    "katsu_cuda_event *": "*mut Event", "katsu_cuda_event **": "*mut *mut Event",
}
RESERVED = {"in", "ref", "type", "fn", "mod", "move", "box", "loop", "match", "use", "where", "self"}


def declarations():
    """[(name, return type, [(argument name, C type)])] in header order."""
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    out = []
    for m in re.finditer(r"(const char \*|int32_t )\s*(katsu_cuda_[a-z0-9_]+)\s*\(([^;]*?)\);", text, flags=re.S):
        args = []
        body = " ".join(m.group(3).split())
        if body != "void":
            for piece in body.split(","):
                piece = piece.strip()
                array = re.match(r"(const )?uint8_t (\w+)\[\w+\]$", piece)
                if array:
                    args.append((array.group(2), "const uint8_t *" if array.group(1) else "uint8_t *"))
                    continue
                name = re.search(r"(\w+)$", piece).group(1)
                ctype = piece[: -len(name)].strip()
                ctype = re.sub(r"\s*\*", " *", ctype).replace("* *", "**")
                args.append((name, ctype))
        out.append((m.group(2), m.group(1).strip(), args))
    return out


def rust_type(ctype):
    if ctype in ("uint8_t *", "const uint8_t *"):
        return "*mut u8" if ctype == "uint8_t *" else "*const u8"
    return TYPES[ctype]


def render():
    constants = re.findall(r"#define (KATSU_[A-Z0-9_]+) (\d+)\b", open(HEADER).read())
    lines = [
        "// GENERATED by gen_ffi.py from include/katsu_cuda.h -- do not edit by hand.",
        "// Not compiled in the repository that carries the kernels: its build image has no Rust toolchain.",
        "#![allow(dead_code)]",
        "use std::os::raw::{c_char, c_void};",
        "",
        "/// Opaque katsu_cuda_ctx: one device, one stream.",
        "#[repr(C)]",
        "pub struct Ctx {",
        "    _private: [u8; 0],",
        "}",
        "/// Opaque katsu_cuda_event.",
        "#[repr(C)]",
        "pub struct Event {",
        "    _private: [u8; 0],",
        "}",
        "",
    ]
    for name, value in constants:
        kind = "usize" if name.endswith("_BYTES") else "i32"
        lines.append(f"pub const {name}: {kind} = {value};")
    lines += ["pub const KATSU_SUM_STATIC_MAX_COUNT: usize = 1 << 30;", "", 'extern "C" {']
    for name, ret, args in declarations():
        rendered = ", ".join(f"{(a + '_') if a in RESERVED else a}: {rust_type(t)}" for a, t in args)
        rust_ret = "*const c_char" if ret.startswith("const char") else "i32"
        lines.append(f"    pub fn {name}({rendered}) -> {rust_ret};")
    lines += ["}", ""]
    return "\n".join(lines)


if __name__ == "__main__":
    text = render()
    if "--check" in sys.argv:
        sys.exit(0 if os.path.exists(OUT) and open(OUT).read() == text else 1)
    with open(OUT, "w") as fh:
        fh.write(text)
    print("wrote", OUT)
