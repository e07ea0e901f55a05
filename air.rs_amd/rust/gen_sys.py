"""Generates airkv-sys/src/lib.rs -- the Rust `extern "C"` declarations of
every function, type and constant in include/air_kv.h -- so the binding and
the header cannot drift apart (tests/test_rust_binding.py checks that the
committed file equals what this script writes).

Run:  python air.rs_amd/rust/gen_sys.py
"""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
HEADER = os.path.join(ROOT, "include", "air_kv.h")
OUT = os.path.join(HERE, "airkv-sys", "src", "lib.rs")

SCALARS = {"int": "c_int", "int32_t": "i32", "int64_t": "i64", "uint32_t": "u32", "uint16_t": "u16",
           "uint64_t": "u64", "uint8_t": "u8", "int8_t": "i8", "size_t": "usize", "float": "f32", "double": "f64",
           "void": "c_void", "char": "c_char"}


def rust_type(ctype: str, opaque: set) -> str:
    t = ctype.strip()
    arr = re.search(r"\[\s*\d*\s*\]$", t)
    if arr:                                   # `uint8_t out[12]` parameters decay to pointers
        t = t[:arr.start()].strip() + " *"
    stars = t.count("*")
    base = t.replace("*", " ").split()
    consts = [i for i, w in enumerate(base) if w == "const"]
    words = [w for w in base if w != "const"]
    name = words[-1] if words else "void"
    inner = SCALARS.get(name, name)
    if stars == 0:
        return inner
    # pointer levels from the inside out: `const T *const *p` is rare here; the
    # first pointer is *const when `const` precedes the base type
    lead_const = bool(consts) and consts[0] == 0
    r = ("*const " if lead_const else "*mut ") + inner
    for _ in range(stars - 1):
        r = ("*const " if "* const" in t or "*const" in t else "*mut ") + r
    return r


def split_params(p: str):
    p = p.strip()
    if p in ("", "void"):
        return []
    return [x.strip() for x in p.split(",")]


def param(decl: str, opaque: set):
    m = re.match(r"(.*?)([A-Za-z_]\w*)\s*(\[\s*\d*\s*\])?$", decl.strip())
    ctype, name, arr = m.group(1), m.group(2), m.group(3) or ""
    if name in ("type", "ref", "self", "fn", "match", "in", "loop", "move"):
        name = name + "_"
    return name, rust_type(ctype + arr, opaque)


def main():
    src = open(HEADER).read()
    body = re.sub(r"/\*.*?\*/", "", src, flags=re.S)
    body = re.sub(r"//[^\n]*", "", body)
    out = ["// Generated by air.rs_amd/rust/gen_sys.py from include/air_kv.h -- do not edit.",
           "//",
           "// Raw bindings of libairkv.so, the C ABI of the MI355X paged KV-cache path.",
           "// This crate is source for Air.rs maintainers; it is not compiled in this",
           "// repository (no Rust toolchain here).  See the safe wrapper in ../airkv.",
           "#![allow(non_camel_case_types, non_upper_case_globals, clippy::all)]",
           "",
           "use core::ffi::{c_char, c_int, c_void};",
           ""]
    for m in re.finditer(r"^#define\s+(AIR_KV_\w+)\s+\(?\s*(-?\w+)\s*(?:<<\s*(\d+))?\s*\)?", body, re.M):
        name, val, sh = m.group(1), m.group(2), m.group(3)
        if name == "AIR_KV_H":
            continue
        v = val.rstrip("uU")
        if sh:
            out.append(f"pub const {name}: usize = {v} << {sh};")
        else:
            out.append(f"pub const {name}: c_int = {v};")
    out.append("")
    opaque = set(re.findall(r"typedef\s+struct\s+(\w+)\s+\1\s*;", body))
    for o in sorted(opaque):
        out.append("#[repr(C)]")
        out.append(f"pub struct {o} {{")
        out.append("    _private: [u8; 0],")
        out.append("}")
        out.append("")
    for m in re.finditer(r"typedef\s+struct\s+(\w+)\s*\{(.*?)\}\s*(\w+)\s*;", body, re.S):
        name, fields = m.group(3), m.group(2)
        out.append("#[repr(C)]")
        out.append("#[derive(Clone, Copy, Debug, Default)]")
        out.append(f"pub struct {name} {{")
        for f in fields.split(";"):
            f = f.strip()
            if not f:
                continue
            fname, ftype = param(f, opaque)
            out.append(f"    pub {fname}: {ftype},")
        out.append("}")
        out.append("")
    for m in re.finditer(r"typedef\s+(\w+)\s*\(\s*\*\s*(\w+)\s*\)\s*\((.*?)\)\s*;", body, re.S):
        ret, name, params = m.group(1), m.group(2), m.group(3)
        ps = ", ".join(param(p, opaque)[1] for p in split_params(params))
        r = SCALARS.get(ret, ret)
        out.append(f"pub type {name} = Option<unsafe extern \"C\" fn({ps}) -> {r}>;")
    out.append("")
    out.append('#[link(name = "airkv")]')
    out.append('extern "C" {')
    decls = re.finditer(r"^\s*((?:const\s+)?[A-Za-z_][\w\s\*]*?)\b(air_[a-z0-9_]+)\s*\(([^;{]*?)\)\s*;", body,
                        re.M | re.S)
    for m in decls:
        ret, name, params = m.group(1).strip(), m.group(2), m.group(3)
        if ret.startswith("typedef"):
            continue
        ps = ", ".join(f"{n}: {t}" for n, t in (param(p, opaque) for p in split_params(" ".join(params.split()))))
        rt = rust_type(ret, opaque)
        out.append(f"    pub fn {name}({ps}){'' if rt == 'c_void' else ' -> ' + rt};")
    out.append("}")
    text = "\n".join(out) + "\n"
    if len(sys.argv) > 1 and sys.argv[1] == "--print":
        sys.stdout.write(text)
        return
    with open(OUT, "w") as f:
        f.write(text)
    print(f"wrote {OUT}")


if __name__ == "__main__":
    main()
