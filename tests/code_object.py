"""The gfx950 code that the library holds, as the CPU tests look at it: its
kernels' metadata and its instructions (by ROCm's llvm-readelf and llvm-objdump)."""
import functools
import os
import re
import shutil
import subprocess
import tempfile
from collections import namedtuple

from arclight_amd import _lib

BIN = os.environ.get("ROCM_LLVM_BIN", "/opt/rocm/llvm/bin")
OBJDUMP, READELF = (os.path.join(BIN, x) for x in ("llvm-objdump", "llvm-readelf"))


def available():
    return all(os.path.exists(x) for x in (_lib.LIB_PATH, OBJDUMP, READELF))


# op: the mnemonic; args: its operands' text; at: address; to: a branch's target or None
Instruction = namedtuple("Instruction", "op args at to")
LINE = re.compile(r"^\s+(?P<op>\S+)(?: (?P<args>.*?))?\s*// (?P<at>[0-9A-F]+):(?: [0-9A-F]{8})+(?: <(?P<sym>\S+?)(?:\+0x(?P<off>[0-9a-f]+))?>)?\s*$")
START = re.compile(r"^([0-9a-f]+) <(\S+)>:$")


def _objects(where):
    shutil.copy(_lib.LIB_PATH, os.path.join(where, "lib"))
    subprocess.run([OBJDUMP, "--offloading", "lib"], cwd=where, check=True, capture_output=True)
    return sorted(os.path.join(where, f) for f in os.listdir(where) if "gfx950" in f)


@functools.lru_cache(None)
def kernels():
    """{name: {field of the kernel's metadata: its number}}."""
    out = {}
    with tempfile.TemporaryDirectory() as where:
        for path in _objects(where):
            text = subprocess.run([READELF, "--notes", path], check=True, capture_output=True, text=True).stdout
            # a kernel's own fields are indented by four, its arguments' deeper
            for part in re.split(r"(?m)^  - (?=\.)", text)[1:]:
                fields = dict(re.findall(r"(?m)^(?:    )?\.(\w+): +(\S+)$", part))
                if "name" in fields:
                    out[fields["name"]] = {k: int(v) for k, v in fields.items() if v.isdigit()}
    return out


@functools.lru_cache(None)
def functions():
    """{name: [Instruction]}, in their order."""
    out = {}
    with tempfile.TemporaryDirectory() as where:
        for path in _objects(where):
            body, starts = None, {}
            text = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", path], check=True, capture_output=True, text=True).stdout
            for line in text.splitlines():
                m = START.match(line)
                if m:
                    starts[m[2]] = int(m[1], 16)
                    body = out.setdefault(m[2], [])
                    continue
                m = LINE.match(line)
                if m and body is not None:
                    to = starts[m["sym"]] + int(m["off"] or "0", 16) if m["sym"] in starts else None
                    body.append(Instruction(m["op"], m["args"] or "", int(m["at"], 16), to))
    return out
