"""Writes the Rust side of the C ABI from include/rustorch_hip.h: one `extern "C"` declaration per exported function,
the `#[repr(C)]` structures and the enum constants, as `src/gpu/hip_ffi.rs` of the reference would hold them (the sibling
of the cudarc bindings behind `CudaKernelExecutor`, src/gpu/cuda_kernels.rs:201-283; feature-off stubs as at :626-700).

    python -m rustorch_amd.ffi_gen            prints the module
    python -m rustorch_amd.ffi_gen --check    exits non-zero when the integration notes at the repository root do not hold the same text

The header is the single source: tests/test_abi.py keeps the integration notes, this generator and the ctypes table in step.
"""
from __future__ import annotations

import re
import sys
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
HEADER = ROOT / "include" / "rustorch_hip.h"
DOC = ROOT / "INTEGRATION.md"
BEGIN, END = "<!-- hip_ffi.rs: generated by python -m rustorch_amd.ffi_gen -->", "<!-- end of hip_ffi.rs -->"

OPAQUE = {"rt_hip_ctx": "RtHipCtx", "rt_hip_qweight": "RtHipQWeight", "rt_hip_llama": "RtHipLlama", "rt_hip_llama_batch": "RtHipLlamaBatch", "rt_hip_event": "RtHipEvent", "rt_hip_paged_kv": "RtHipPagedKv"}
STRUCTS = {"rt_hip_devinfo": "RtHipDevInfo", "rt_hip_llama_config": "RtHipLlamaConfig"}
SCALARS = {"int": "i32", "float": "f32", "double": "f64", "size_t": "usize", "uint64_t": "u64", "uint16_t": "u16", "int8_t": "i8", "uint8_t": "u8",
           "char": "std::os::raw::c_char", "void": "std::ffi::c_void"}


def strip_comments(text: str) -> str:
    return re.sub(r"/\*.*?\*/", " ", text, flags=re.S)


def rust_type(ctype: str) -> str:
    """`const float *const *` -> `*const *const f32` (pointer levels read right to left)."""
    tokens = re.findall(r"\*|\w+", ctype)
    base, levels, pending_const = None, [], False
    for t in tokens:
        if t == "const":
            if base is None:
                pending_const = True
            else:
                levels[-1] = True          # `* const`: the pointer itself is const -- irrelevant to Rust's pointee mutability
            continue
        if t == "*":
            levels.append(False)
            continue
        base = t
    base_const = pending_const
    if base in OPAQUE:
        r = OPAQUE[base]
    elif base in STRUCTS:
        r = STRUCTS[base]
    else:
        r = SCALARS[base]
    # innermost pointee constness comes from the base; an outer level points at a pointer declared `*const` in C when
    # that pointer was followed by `const`
    n = len(levels)
    if n == 0:
        return r
    out = ("*const " if base_const else "*mut ") + r
    for i in range(1, n):
        out = ("*const " if levels[i - 1] else "*mut ") + out
    return out


def functions(text: str):
    """[(name, return type, [(arg name, arg type)])] in header order."""
    out = []
    for ret, name, args in re.findall(r"RT_HIP_API\s+([\w\s\*]+?)\b(rt_\w+)\s*\(([^;]*?)\)\s*;", strip_comments(text)):
        params = []
        if args.strip() != "void":
            for a in args.split(","):
                m = re.match(r"\s*(.*?)(\w+)\s*$", a.replace("\n", " "))
                params.append((m.group(2), m.group(1).strip()))
        out.append((name, ret.strip(), params))
    return out


def struct_fields(text: str, cname: str):
    body = re.search(r"typedef struct \{([^{}]*)\}\s*%s\s*;" % cname, strip_comments(text)).group(1)
    fields = []
    for decl in body.split(";"):
        decl = decl.strip()
        if not decl:
            continue
        ctype, names = decl.split(None, 1)
        for nm in names.split(","):
            nm = nm.strip()
            arr = re.match(r"(\w+)\[(\d+)\]", nm)
            if arr:
                fields.append((arr.group(1), "[%s; %s]" % (SCALARS[ctype], arr.group(2))))
            else:
                fields.append((nm, SCALARS[ctype]))
    return fields


def enum_values(text: str, cname: str):
    body = re.search(r"typedef enum \{([^{}]*)\}\s*%s\s*;" % cname, strip_comments(text)).group(1)
    return [(k, int(v)) for k, v in re.findall(r"(\w+)\s*=\s*(\d+)", body)]


RUST_KEYWORDS = {"type", "ref", "in", "out_ref", "move", "fn", "mod", "box", "final"}


def generate() -> str:
    text = HEADER.read_text()
    lines = ["// src/gpu/hip_ffi.rs -- generated from include/rustorch_hip.h by `python -m rustorch_amd.ffi_gen`; do not edit.",
             "#![allow(non_camel_case_types, dead_code)]", ""]
    for c, r in OPAQUE.items():
        lines.append("#[repr(C)] pub struct %s { _private: [u8; 0] }      // %s" % (r, c))
    lines.append("")
    for c, r in STRUCTS.items():
        lines.append("#[repr(C)] #[derive(Clone, Copy)]")
        lines.append("pub struct %s {      // %s" % (r, c))
        for nm, ty in struct_fields(text, c):
            lines.append("    pub %s: %s," % (nm, ty))
        lines.append("}")
    lines.append("")
    for cname in ("rt_hip_status", "rt_ggml_type", "rt_hip_rope", "rt_hip_llama_slot"):
        for k, v in enum_values(text, cname):
            lines.append("pub const %s: i32 = %d;" % (k, v))
        lines.append("")
    fns = functions(text)
    lines.append("#[cfg(feature = \"hip\")]")
    lines.append("#[link(name = \"rustorch_hip\", kind = \"static\")]")
    lines.append("extern \"C\" {")
    for name, ret, params in fns:
        args = ", ".join("%s: %s" % (p + "_" if p in RUST_KEYWORDS else p, rust_type(t)) for p, t in params)
        lines.append("    pub fn %s(%s) -> %s;" % (name, args, rust_type(ret)))
    lines.append("}")
    lines.append("")
    lines.append("// With the feature off every entry point is a stub that reports the missing backend, the form the CUDA executor's")
    lines.append("// stubs take (src/gpu/cuda_kernels.rs:626-700): callers get RT_HIP_ERR_NO_DEVICE and map it to DeviceNotAvailable.")
    lines.append("#[cfg(not(feature = \"hip\"))]")
    lines.append("mod disabled {")
    lines.append("    use super::*;")
    for name, ret, params in fns:
        args = ", ".join("_%s: %s" % (p, rust_type(t)) for p, t in params)
        rt = rust_type(ret)
        if rt == "i32":
            body = "0" if name == "rt_hip_device_count" else "RT_HIP_ERR_NO_DEVICE"
        elif rt == "usize":
            body = "0"
        else:
            body = "b\"rustorch was built without the hip feature\\0\".as_ptr() as %s" % rt
        lines.append("    pub unsafe fn %s(%s) -> %s { %s }" % (name, args, rt, body))
    lines.append("}")
    lines.append("#[cfg(not(feature = \"hip\"))]")
    lines.append("pub use disabled::*;")
    return "\n".join(lines) + "\n"


def doc_block() -> str:
    """The generated module as the integration notes hold it (between the two marker comments)."""
    text = DOC.read_text()
    a, b = text.index(BEGIN), text.index(END)
    inner = text[a + len(BEGIN):b]
    m = re.search(r"```rust\n(.*?)```", inner, flags=re.S)
    return m.group(1)


def main(argv) -> int:
    if "--check" in argv:
        if doc_block() != generate():
            print("%s does not hold what the header generates; run python -m rustorch_amd.ffi_gen --write" % DOC.name, file=sys.stderr)
            return 1
        return 0
    if "--write" in argv:
        text = DOC.read_text()
        a, b = text.index(BEGIN), text.index(END)
        DOC.write_text(text[:a + len(BEGIN)] + "\n```rust\n" + generate() + "```\n" + text[b:])
        return 0
    sys.stdout.write(generate())
    return 0


if __name__ == "__main__":
    sys.exit(main(sys.argv[1:]))
