"""The compiled kernels of liblsamp.so as text: what each needs of the device, and its
instructions, for tests of what inline assembly leaves to its author."""
from __future__ import annotations

import functools
import os
import re
import struct
import subprocess
import tempfile
from typing import Dict, Iterator, List, NamedTuple, Tuple

LLVM = "/opt/rocm/llvm/bin"
MAGIC = b"__CLANG_OFFLOAD_BUNDLE__"


def code_objects(library: str) -> Iterator[bytes]:
    """The library's code objects for the device, one a source file."""
    with open(library, "rb") as f:
        data = f.read()
    at = data.find(MAGIC)
    while at >= 0:
        count, = struct.unpack_from("<Q", data, at + len(MAGIC))
        place, found = at + len(MAGIC) + 8, False
        for _ in range(min(count, 16)):
            offset, size, name = struct.unpack_from("<QQQ", data, place)
            triple = data[place + 24:place + 24 + name]
            place += 24 + name
            if b"amdgcn" in triple and size:
                found = True
                yield data[at + offset:at + offset + size]
        at = data.find(MAGIC, at + (len(MAGIC) if found else 1))


def _run(tool: str, *args: str) -> str:
    return subprocess.run([os.path.join(LLVM, tool), *args], check=True, capture_output=True,
                          text=True).stdout


def scratch_bytes(library: str) -> Dict[str, int]:
    """Bytes of scratch memory a thread, for each kernel (mangled names)."""
    out = {}
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "code")
        for code in code_objects(library):
            with open(path, "wb") as f:
                f.write(code)
            name = None
            for line in _run("llvm-readelf", "--notes", path).splitlines():
                m = re.match(r"\s+(?:- )?\.(name|private_segment_fixed_size):\s+(\S+)", line)
                if not m:
                    continue
                # (an argument's name is indented further, and no kernel's)
                if m[1] == "name" and m[2].startswith("_Z"):
                    name = m[2]
                elif m[1] == "private_segment_fixed_size":
                    out[name] = int(m[2])
    return out


class Instruction(NamedTuple):
    op: str
    args: Tuple[str, ...]
    branch: int  # the address it goes to, or -1


class Function(NamedTuple):
    name: str
    code: List[Instruction]
    before: List[List[int]]  # the places an instruction may be reached from


@functools.lru_cache(maxsize=1)
def _texts(library: str) -> List[Tuple[str, str]]:
    """Every function's name and instructions."""
    out = []
    with tempfile.TemporaryDirectory() as d:
        path = os.path.join(d, "code")
        for code in code_objects(library):
            with open(path, "wb") as f:
                f.write(code)
            text = _run("llvm-objdump", "-d", "--no-show-raw-insn", path)
            for part in re.split(r"\n(?=[0-9a-f]{16} <)", text):
                head = re.match(r"[0-9a-f]{16} <(.*)>:\n", part)
                if head:
                    out.append((head[1], part[head.end():]))
    return out


def functions(library: str, having: str, named: str = "") -> Iterator[Function]:
    """The functions of the code objects that have an instruction named `having`, and `named`
    in their own names."""
    for name, text in _texts(library):
        if having in text and named in name:
            yield _function(name, text)


def _function(name: str, text: str) -> Function:
    code, places = [], {}
    for line in text.splitlines():
        m = re.match(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+):?\s*(?:<.*\+0x([0-9a-f]+)>)?", line)
        if not m:
            continue
        places[int(m[3], 16)] = len(code)
        to = int(m[4], 16) if m[4] and "branch" in m[1] else -1
        code.append(Instruction(m[1], tuple(a.strip() for a in m[2].split(",")), to))
    first = min(places) if places else 0
    before = [[] for _ in code]
    for i, c in enumerate(code):
        next_ = [] if c.op in ("s_endpgm", "s_branch", "s_setpc_b64") else [i + 1]
        if c.branch >= 0:
            next_.append(places[first + c.branch])
        for n in next_:
            if n < len(code):
                before[n].append(i)
    return Function(name, code, before)


def registers(arg: str, kind: str) -> range:
    """The scalar (kind "s") or vector ("v") registers that an operand names."""
    m = re.match(kind + r"\[(\d+):(\d+)\]$|" + kind + r"(\d+)$", arg.split(" ")[0])
    if not m:
        return range(0)
    return range(int(m[3]), int(m[3]) + 1) if m[3] else range(int(m[1]), int(m[2]) + 1)


def waits(c: Instruction) -> int:
    """Wait states that an instruction is worth to those behind it."""
    return int(c.args[0], 0) + 1 if c.op == "s_nop" else 1


def scalar_results(c: Instruction) -> List[int]:
    """Scalar registers that a vector instruction writes."""
    if not c.op.startswith("v_"):
        return []
    return [r for a in c.args[:2 if "_co_" in c.op or "div_scale" in c.op else 1]
            for r in registers(a, "s")]


def _overlap(a: range, b) -> bool:
    return any(r in a for r in b)


def stale_addresses(f: Function, op: str = "global_load_lds", states: int = 5) -> List[int]:
    """Places of memory instructions that read a scalar register which a vector instruction
    wrote fewer than `states` wait states before, on any path."""
    bad = []
    for i, c in enumerate(f.code):
        if not c.op.startswith(op):
            continue
        reads = [r for a in c.args for r in registers(a, "s")]
        if not reads:
            continue
        todo, seen = [(i, 0)], set()
        while todo:
            at, passed = todo.pop()
            for b in f.before[at]:
                if (b, passed) in seen:
                    continue
                seen.add((b, passed))
                if _overlap(range(min(reads), max(reads) + 1), scalar_results(f.code[b])):
                    bad.append(i)
                    todo = []
                    break
                total = passed + waits(f.code[b])
                if total < states:
                    todo.append((b, total))
    return bad


def unsettled_stores(f: Function, flags: Tuple[str, ...], states: int = 2) -> Tuple[int, List[int]]:
    """The number of stores of 128 bits with these flags, and the places of those that no wait
    of `states` wait states follows at once: a vector instruction may overwrite their data, if
    not here then after any change of the code around them."""
    stores = [i for i, c in enumerate(f.code)
              if c.op == "global_store_dwordx4" and set(c.args[-1].split()) == {"off", *flags}]
    return len(stores), [i for i in stores if f.code[i + 1].op != "s_nop"
                         or waits(f.code[i + 1]) < states]
