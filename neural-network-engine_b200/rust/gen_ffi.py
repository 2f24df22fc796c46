"""Generates src/gpu/cuda/ffi.rs from include/nne_cuda.h: one `extern "C"` declaration per exported
symbol, the status codes, the opaque handle types and the plan item struct.  Run from anywhere:

    python neural-network-engine_b200/rust/gen_ffi.py            # rewrites ffi.rs
    python neural-network-engine_b200/rust/gen_ffi.py --check    # exit 1 if ffi.rs is out of date

The CPU test-suite runs the same generator and compares, so the Rust bindings cannot drift from
the header."""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
HEADER = os.path.join(HERE, "..", "..", "include", "nne_cuda.h")
OUT = os.path.join(HERE, "src", "gpu", "cuda", "ffi.rs")

SCALARS = {"int": "c_int", "unsigned int": "c_uint", "size_t": "usize", "float": "f32", "int8_t": "i8",
           "uint8_t": "u8", "int32_t": "i32", "double": "f64", "uint64_t": "u64", "void": "c_void", "char": "c_char"}
OPAQUE = ["nne_ctx", "nne_qlinear", "nne_qlinear4", "nne_kv_cache", "nne_plan", "nne_shard_group"]


def rust_type(c: str) -> str:
    """C parameter or return type (without the name) -> Rust."""
    c = " ".join(c.replace("*", " * ").split())
    parts = c.split(" * ")
    stars = c.count("*")
    if stars == 0:
        base = c.replace("const ", "").strip()
        return SCALARS.get(base, base)
    # walk from the base outwards: each '*' takes the constness of what precedes it
    tokens = c.split(" ")
    base_tokens, i = [], 0
    while tokens[i] != "*":
        base_tokens.append(tokens[i])
        i += 1
    const = "const" in base_tokens
    base = " ".join(t for t in base_tokens if t != "const")
    ty = SCALARS.get(base, base)
    while i < len(tokens):
        assert tokens[i] == "*", c
        ty = ("*const " if const else "*mut ") + ty
        const = False
        i += 1
        if i < len(tokens) and tokens[i] == "const":
            const = True
            i += 1
    return ty


def parse(header_text: str):
    text = re.sub(r"/\*.*?\*/", "", header_text, flags=re.S)
    funcs = []
    for m in re.finditer(r"NNE_API\s+([\w\s\*]+?)\b(nne_\w+)\s*\(([^;]*?)\)\s*;", text, flags=re.S):
        ret, name, params = " ".join(m.group(1).split()), m.group(2), " ".join(m.group(3).split())
        args = []
        if params != "void":
            for p in params.split(","):
                p = p.strip()
                pm = re.match(r"(.*?)(\w+)$", p)
                args.append((pm.group(2), rust_type(pm.group(1).strip())))
        funcs.append((name, rust_type(ret), args))
    structs = []
    for m in re.finditer(r"typedef struct (nne_\w+) \{(.*?)\} \1;", text, flags=re.S):
        fields = []
        for f in m.group(2).split(";"):
            fm = re.match(r"(.*?)(\w+)$", " ".join(f.split()))
            if fm:
                fields.append((fm.group(2), rust_type(fm.group(1).strip())))
        if m.group(1) != "nne_plan_item":  # written out below, with its own comment
            structs.append((m.group(1), fields))
    statuses = re.findall(r"(NNE_(?:OK|ERR_\w+))\s*=\s*(\d+)", text)
    inputs = re.findall(r"(NNE_INPUT_\w+|NNE_B?F16)\s*=\s*(\d+)", text)
    handle_bytes = re.search(r"#define\s+NNE_SHARD_HANDLE_BYTES\s+(\d+)", text).group(1)
    return funcs, statuses, inputs, handle_bytes, structs


def generate(header_text: str) -> str:
    funcs, statuses, inputs, handle_bytes, structs = parse(header_text)
    out = ["//! Raw bindings of `include/nne_cuda.h`: one declaration per exported symbol, nothing else.",
           "//! GENERATED by `gen_ffi.py` from the header - edit the header, then run the generator.",
           "#![allow(non_camel_case_types)]",
           "use std::os::raw::{c_char, c_int, c_uint, c_void};", ""]
    for h in OPAQUE:
        out += ["#[repr(C)]", f"pub struct {h} {{", "    _private: [u8; 0],", "}"]
    out += ["", "/// One forward of a fused plan (`nne_plan_item`).", "#[repr(C)]", "#[derive(Clone, Copy)]",
            "pub struct nne_plan_item {", "    pub layer: *mut nne_qlinear,", "    pub x: *const f32,",
            "    pub y: *mut f32,", "    pub input_op: c_int,", "    pub eps: f32,", "    pub gamma: *const f32,",
            "    pub x2: *const f32,", "    pub residual: *const f32,", "}", ""]
    for name, fields in structs:
        out += [f"/// `{name}`.", "#[repr(C)]", "#[derive(Clone, Copy)]", f"pub struct {name} {{"]
        out += [f"    pub {f}: {t}," for f, t in fields] + ["}", ""]
    for name, val in statuses + inputs:
        out.append(f"pub const {name}: c_int = {val};")
    out += [f"pub const NNE_SHARD_HANDLE_BYTES: usize = {handle_bytes};", "", 'extern "C" {']
    for name, ret, args in funcs:
        arglist = ", ".join(f"{a}: {t}" for a, t in args)
        line = f"    pub fn {name}({arglist}) -> {ret};"
        if len(line) > 110:
            body = "".join(f"        {a}: {t},\n" for a, t in args)
            line = f"    pub fn {name}(\n{body}    ) -> {ret};"
        out.append(line)
    out += ["}", ""]
    return "\n".join(out)


def main():
    text = generate(open(HEADER).read())
    if "--check" in sys.argv:
        same = os.path.exists(OUT) and open(OUT).read() == text
        print("ffi.rs is up to date" if same else "ffi.rs is OUT OF DATE: run gen_ffi.py")
        sys.exit(0 if same else 1)
    os.makedirs(os.path.dirname(OUT), exist_ok=True)
    open(OUT, "w").write(text)
    print("wrote", OUT)


if __name__ == "__main__":
    main()
