"""The Rust side of the 8-bit serving operators: structs as the header declares them, every entry point wrapped."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _read(*path):
    with open(os.path.join(ROOT, *path)) as f:
        return f.read()


def test_paged_structs_list_the_header_fields_in_order():
    from rmlk_amd import _lib
    header = re.sub(r"/\*.*?\*/", " ", _read("include", "rmlk_hip.h"), flags=re.S)
    ffi = _read("hip", "src", "ffi.rs")
    for name, mirror in (("rmlk_paged_cache", _lib.PagedCacheStruct), ("rmlk_paged_batch", _lib.PagedBatchStruct)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), header, flags=re.S).group(1)
        decls = [d.split() for d in body.replace("*", " * ").split(";") if d.strip()]
        fields = [d[-1] for d in decls]
        rust = re.search(r"pub struct %s \{(.*?)\n\}" % name, ffi, flags=re.S).group(1)
        assert re.findall(r"pub (\w+):", rust) == fields
        assert [n for n, _ in mirror._fields_] == fields
        # integers of the same width on all three sides
        width = {"int32_t": 4, "int64_t": 8}
        types = dict(re.findall(r"pub (\w+): ([^,]+),", rust))
        for d in decls:
            size = 8 if "*" in d else width[d[0]]
            assert getattr(mirror, d[-1]).size == size, (name, d[-1])
            assert {"i32": 4, "i64": 8}.get(types[d[-1]], 8) == size, (name, d[-1])


def test_every_entry_point_is_wrapped():
    text = _read("hip", "src", "kernels", "int8.rs") + _read("hip", "src", "kernels", "paged.rs")
    for name in ("quantize_rows", "rmsnorm_quantize_rows", "matmul_int8", "matmul_int8_workspace_size", "paged_append",
                 "paged_attention", "paged_attention_workspace_size"):
        assert f"ffi::rmlk_hip_{name}(" in text, name
    mods = _read("hip", "src", "kernels", "mod.rs")
    assert "pub mod int8;" in mods and "pub mod paged;" in mods
