"""Writes src/ffi.rs, the raw `extern "C"` declarations of
libatlas_hip_ops.so, from include/atlas_hip_ops.h and include/atlas_gguf.h
(one declaration per C entry point, in header order).  Run after changing a
header: `python crates/atlas-hip-ops/gen_ffi.py`; tests/test_rust_crate.py
checks that the committed file still matches the headers."""
import os
import re
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))
HEADERS = [os.path.join(ROOT, "include", h) for h in ("atlas_hip_ops.h", "atlas_gguf.h")]

SCALARS = {"int": "c_int", "float": "f32", "double": "f64", "size_t": "usize", "uint8_t": "u8", "uint16_t": "u16",
           "uint32_t": "u32", "uint64_t": "u64", "int64_t": "i64", "char": "c_char", "void": "c_void",
           "atlas_hip_ctx": "AtlasHipCtx", "atlas_gguf": "AtlasGguf", "atlas_gguf_tensor": "AtlasGgufTensor",
           "atlas_dispatch_timing": "AtlasDispatchTiming", "atlas_hip_telemetry": "AtlasHipTelemetry",
           "atlas_paged_cache": "AtlasPagedCache"}


def declarations(path):
    """(return type, name, [(type, name)]) of every function prototype."""
    text = re.sub(r"/\*.*?\*/", "", open(path).read(), flags=re.S)
    text = re.sub(r"#.*", "", text)
    out = []
    for m in re.finditer(r"([A-Za-z_][\w \*]*?)\b(atlas_\w+)\s*\(([^;{]*?)\)\s*;", text, flags=re.S):
        ret, name, params = " ".join(m.group(1).split()), m.group(2), " ".join(m.group(3).split())
        args = []
        if params and params != "void":
            for p in params.split(","):
                p = p.strip()
                pm = re.match(r"(.*?)(\w+)$", p)
                args.append((" ".join(pm.group(1).replace("*", " * ").split()), pm.group(2)))
        out.append((ret, name, args))
    return out


def rust_type(c):
    """C type text -> Rust FFI type ('const float *' -> '*const f32')."""
    toks = c.replace("*", " * ").split()
    const_first = toks and toks[0] == "const"
    if const_first:
        toks = toks[1:]
    base, stars = toks[0], toks.count("*")
    if base not in SCALARS:
        raise SystemExit(f"unmapped C type: {c}")
    t = SCALARS[base]
    for i in range(stars):
        # the const of `const T *` qualifies the innermost pointee
        t = f"*{'const' if (const_first and i == 0) else 'mut'} {t}"
    return t


KEYWORDS = {"type", "ref", "in", "fn", "loop", "match", "move", "mod", "self", "super", "use", "where", "box"}


def render():
    lines = ["// Generated by crates/atlas-hip-ops/gen_ffi.py from include/atlas_hip_ops.h and",
             "// include/atlas_gguf.h; do not edit by hand.  Raw declarations of",
             "// libatlas_hip_ops.so: every pointer is a device pointer unless the header",
             "// says otherwise (the atlas_ops_* host-slice entry points take host memory).",
             "#![allow(non_camel_case_types, dead_code)]", "",
             "use std::os::raw::{c_char, c_int, c_void};", "",
             "#[repr(C)]", "pub struct AtlasHipCtx {", "    _private: [u8; 0],", "}", "",
             "#[repr(C)]", "pub struct AtlasGguf {", "    _private: [u8; 0],", "}", "",
             "/// atlas_dispatch_timing (DispatchTiming, crates/atlas-metal/src/lib.rs:81-88).",
             "#[repr(C)]", "#[derive(Debug, Default, Clone, Copy)]",
             "pub struct AtlasDispatchTiming {", "    pub wall_ms: f64,", "    pub gpu_ms: f64,", "}", "",
             "/// atlas_hip_telemetry (RuntimeTelemetry, crates/atlas-metal/src/lib.rs:91-193).",
             "#[repr(C)]", "#[derive(Debug, Default, Clone, Copy)]", "pub struct AtlasHipTelemetry {",
             "    pub dispatches: u64,", "    pub syncs: u64,", "    pub upload_bytes: u64,",
             "    pub readback_bytes: u64,", "    pub allocations: u64,", "    pub resident_bytes: u64,",
             "    pub peak_resident_bytes: u64,", "}", "",
             "/// atlas_paged_cache (no counterpart in the reference).",
             "#[repr(C)]", "#[derive(Debug, Clone, Copy)]", "pub struct AtlasPagedCache {",
             "    pub pages: *mut c_void,", "    pub page_table: *const u32,", "    pub page_count: u32,",
             "    pub page_size: u32,", "    pub kv_heads: u32,", "    pub head_dim: u32,", "    pub sequences: u32,",
             "    pub table_width: u32,", "    pub format: c_int,", "}", "",
             "/// atlas_gguf_tensor (GgufTensor, crates/atlas-core/src/gguf.rs:80-87).",
             "#[repr(C)]", "#[derive(Debug, Clone, Copy)]", "pub struct AtlasGgufTensor {",
             "    pub name: *const c_char,", "    pub name_len: u64,", "    pub n_dims: u32,", "    pub dims: [u64; 4],",
             "    pub type_: u32,", "    pub offset: u64,", "    pub bytes: u64,", "}", "",
             "pub const ATLAS_OK: c_int = 0;", "pub const ATLAS_ERR_NO_DEVICE: c_int = -1;",
             "pub const ATLAS_ERR_INVALID_INPUT: c_int = -2;", "pub const ATLAS_ERR_COMMAND_FAILED: c_int = -3;",
             "pub const ATLAS_ERR_OUT_OF_MEMORY: c_int = -4;", "",
             "pub const ATLAS_REDUCTION_SEQUENTIAL: c_int = 0;", "pub const ATLAS_REDUCTION_WIDE: c_int = 1;",
             "pub const ATLAS_REDUCTION_AUTO: c_int = 2;", "",
             "pub const ATLAS_GGUF_F32: u32 = 0;", "pub const ATLAS_GGUF_F16: u32 = 1;",
             "pub const ATLAS_GGUF_Q4_0: u32 = 2;", "pub const ATLAS_GGUF_Q8_0: u32 = 8;",
             "pub const ATLAS_GGUF_Q6_K: u32 = 14;", "",
             "#[link(name = \"atlas_hip_ops\")]", "extern \"C\" {"]
    for path in HEADERS:
        lines.append(f"    // {os.path.relpath(path, ROOT)}")
        for ret, name, args in declarations(path):
            params = ", ".join(f"{a if a not in KEYWORDS else a + '_'}: {rust_type(t)}" for t, a in args)
            r = "" if ret == "void" else f" -> {rust_type(ret)}"
            lines.append(f"    pub fn {name}({params}){r};")
    lines += ["}", ""]
    return "\n".join(lines)


if __name__ == "__main__":
    target = os.path.join(HERE, "src", "ffi.rs")
    text = render()
    if len(sys.argv) > 1 and sys.argv[1] == "--check":
        sys.exit(0 if open(target).read() == text else 1)
    open(target, "w").write(text)
    print(f"wrote {target}")
