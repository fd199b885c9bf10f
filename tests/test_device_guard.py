"""Every entry point of the library launches, copies and allocates on its handle's device, whatever the caller's current device is, and
leaves the caller's as it was.  With one GPU no call can show it, so the source is read: each function of titan_kv.cu that makes a CUDA
call or a launch constructs OnDevice before the first of them."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "titan_engine_b200", "csrc", "titan_kv.cu")

# reached only from functions that hold the guard
GUARDED_BY_CALLER = {"run_evictions", "prefetch_layer", "multi_workspace", "workspace_alloc"}
# takes no handle: the caller's current device is the one that is meant
NO_HANDLE = {"tk_combine_partials"}
HARMLESS = ("cudaGetErrorString", "cudaGetDevice")
USE = re.compile(r"\b(cuda[A-Z]\w*|tk::launch_\w+|tk::make_\w+_maps?)\s*\(")


def functions(text):
    """(name, body) of the functions defined at file or namespace level."""
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)
    text = re.sub(r'"(\\.|[^"\\\n])*"', '""', text)
    text = re.sub(r"#define(\\\n|[^\n])*", "", text)
    out, at = [], 0
    head = re.compile(r"^[ \t]*(?:static |inline )*[\w:*& <>]+?[ *&](\w+)\(([^;{}]*)\)\s*(?:const\s*)?\{", re.M)
    while True:
        m = head.search(text, at)
        if not m:
            return out
        depth, i = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[i], 0)
            i += 1
        out.append((m.group(1), text[m.end():i]))
        at = i


def test_every_function_that_touches_the_device_holds_the_guard():
    found = functions(open(SOURCE).read())
    names = [n for n, _ in found]
    for known in ("tk_kv_seq_fork", "step_begin_impl", "tk_kv_decode_exchange", "tk_kv_read", "tk_kv_append", "host_flush"):
        assert known in names, known                        # the parser sees what it should
    bare = []
    for name, body in found:
        if name in GUARDED_BY_CALLER | NO_HANDLE | {"OnDevice"}:
            continue
        uses = [m.start() for m in USE.finditer(body) if m.group(1) not in HARMLESS]
        guard = body.find("OnDevice ")
        if uses and (guard < 0 or guard > uses[0]):
            bare.append(name)
    assert not bare, bare


def test_the_current_device_is_set_by_the_guard_alone():
    for name, body in functions(open(SOURCE).read()):
        if name != "OnDevice":
            assert "cudaSetDevice" not in body, name
