"""The Rust declarations that INTEGRATION.md gives a host, against the C header: the same functions, argument for argument."""
import os
import re

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TYPES = {"void*": "*mut c_void", "const void*": "*const c_void", "int32_t": "i32", "size_t": "usize", "float": "f32", "uint64_t": "u64",
         "int32_t*": "*mut i32", "const int32_t*": "*const i32", "float*": "*mut f32", "const float*": "*const f32",
         "uint32_t*": "*mut u32", "const uint32_t*": "*const u32", "rt_err_detail*": "*mut RtErrDetail", "int": "c_int"}


def read(name):
    with open(os.path.join(ROOT, name)) as f:
        return f.read()


def prototypes(text):
    """{name: (result, [argument types])} of the header's functions, as written in Rust where the type is a plain one."""
    text = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    out = {}
    for result, name, args in re.findall(r"^(int|size_t|void \*|void|const char \*)\s*(rt_\w+)\(([^;{]*)\);", text, re.M):
        types = []
        for a in [] if args.strip() == "void" else args.split(","):
            c = re.match(r"(.*?)\s*(\w+)$", " ".join(a.split())).group(1).replace(" *", "*")
            types.append(TYPES.get(c, c))
        out[name] = result.replace(" ", ""), types
    return out


def declarations(text):
    out = {}
    for name, args, result in re.findall(r"pub fn (rt_\w+)\(([^)]*)\)(?: -> ([^;]+))?;", text):
        out[name] = (result or "").strip(), [a.split(":", 1)[1].strip() for a in " ".join(args.split()).rstrip(", ").split(", ") if a]
    return out


HEADER, RUST = prototypes(read("include/rt_attn.h")), declarations(read("INTEGRATION.md"))


def test_what_is_declared_is_what_the_header_has():
    assert len(HEADER) > 50 and len(RUST) > 20
    for name, (_, args) in RUST.items():
        assert name in HEADER, name
        assert len(args) == len(HEADER[name][1]), name
        for got, want in zip(args, HEADER[name][1]):
            assert got == want or want not in TYPES.values(), (name, got, want)


def test_the_entries_of_small_caches_are_all_declared():
    text = read("include/rt_attn.h")
    section = text[text.index("caches that are kept small:"):text.index("---- device buffers")]
    names = set(prototypes(section))
    assert len(names) == 12 and names <= set(RUST), names - set(RUST)
    for name in names:
        assert RUST[name] == ({"int": "c_int", "size_t": "usize"}[HEADER[name][0]], HEADER[name][1]), name
