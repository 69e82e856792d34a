"""Build libitts_hip.so in-tree with hipcc for gfx950 (no cmake/ninja needed).

Each ``csrc/*.hip`` compiles to its own object (in parallel, only when it or a header changed),
then one ``hipcc -shared`` link.  Used by ``__graft_entry__.build()``; also runnable as
``python -m indextts._build [--force]``.  ``ITTS_HIPCC_DEFS="-DX=1 ..."`` and ``ITTS_BUILD_OUT=path``
build an experiment variant next to the product library (microbenchmarks load it via
``ITTS_HIP_LIB``).
"""
from __future__ import annotations

import glob
import os
import re
import shlex
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(PKG_DIR), "csrc")
INCLUDE = os.path.join(os.path.dirname(os.path.dirname(PKG_DIR)), "include")
OUT = os.path.join(PKG_DIR, "libitts_hip.so")
ARCH = os.environ.get("PYTORCH_ROCM_ARCH", "gfx950")
# -packed-fp32-ops: no v_pk_{add,mul,fma}_f32, which hipcc -O3 forms from ordinary float code by itself (the
# host pass warns that it does not know the feature: harmless)
FLAGS = ["-O3", "-std=c++17", "-fPIC", "-Wno-unused-result",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def sources():
    return sorted(glob.glob(os.path.join(CSRC, "*.hip")))


def _headers():
    return glob.glob(os.path.join(CSRC, "*.h")) + glob.glob(os.path.join(INCLUDE, "*.h"))


def needs_rebuild(out: str = OUT) -> bool:
    if not os.path.exists(out):
        return True
    t = os.path.getmtime(out)
    return any(os.path.getmtime(s) > t for s in sources() + _headers())


# ---- matrix products written as inline assembly (csrc/fp8_linear.hip) ----
# The compiler does not know them as matrix instructions, so it puts no waits between a vector instruction that writes an operand and
# the product, nor around a copy of the sums, which it may place anywhere.  That the kernel holds neither is a property of its
# assembly, looked at whenever the file is compiled.
CHECKED = {"fp8_linear.hip": "fp8_linear_large_kernel"}
WAIT = 4  # issue slots between a vector write and the product that reads it (two are needed)


def _registers(operand):
    m = re.fullmatch(r"([va])\[(\d+):(\d+)\]", operand)
    if m:
        return {m[1] + str(i) for i in range(int(m[2]), int(m[3]) + 1)}
    return {operand} if re.fullmatch(r"[va]\d+", operand) else set()


def check_products(text: str, kernel: str) -> int:
    """The number of products in the functions of the assembly whose name holds ``kernel``; RuntimeError where one may read a
    vector register too early, or where anything but a product touches a sum between the first and the last."""
    count = 0
    for name, body in re.findall(r"^(\w*%s\w*):(.*?)^\.Lfunc_end" % kernel, text, re.M | re.S):
        code, label, jumps = [], {}, {}  # instructions as (name, operands); label -> index of the next one, and of jumps to it
        for line in body.split("\n"):
            line = line.split(";")[0].strip()
            if line.startswith(".LBB"):
                label[line.rstrip(":")] = len(code)
            elif line and not line.startswith("."):
                op, _, rest = line.partition(" ") if " " in line else line.partition("\t")
                operands = [o.strip().split(" ")[0] for o in rest.split(",")]
                if op.startswith(("s_cbranch", "s_branch")):
                    jumps.setdefault(operands[0], []).append(len(code))
                code.append((op, operands))
        into = {}
        for at, froms in ((label[k], v) for k, v in jumps.items()):
            into.setdefault(at, []).extend(froms)
        products = [i for i, (op, _) in enumerate(code) if op.startswith("v_mfma")]
        count += len(products)
        for i in products:
            reads = set().union(*(_registers(o) for o in code[i][1][1:]))
            todo, seen = [(i, WAIT)], set()
            while todo:
                at, left = todo.pop()
                if left <= 0 or (at, left) in seen:
                    continue
                seen.add((at, left))
                todo += [(j, left - 1) for j in into.get(at, ())]
                if at == 0 or code[at - 1][0] in ("s_branch", "s_endpgm"):
                    continue
                op, operands = code[at - 1]
                if op.startswith("v_") and not op.startswith("v_mfma") and _registers(operands[0]) & reads:
                    raise RuntimeError(f"{name}: {op} {', '.join(operands)} right before the product that reads it")
                todo.append((at - 1, left - (1 + int(operands[0], 0) if op == "s_nop" else 1)))
        for op, operands in code[products[0]:products[-1]] if products else ():
            if not op.startswith("v_mfma") and any(r[0] == "a" for o in operands for r in _registers(o)):
                raise RuntimeError(f"{name}: {op} {', '.join(operands)} among the products")
    return count


def build(force: bool = False, verbose: bool = True, out: str = None) -> str:
    out = out or os.environ.get("ITTS_BUILD_OUT", OUT)
    defs = shlex.split(os.environ.get("ITTS_HIPCC_DEFS", ""))
    if not force and not needs_rebuild(out):
        return out
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    tag = "".join(c if c.isalnum() else "_" for c in " ".join(defs))[:80] or "default"
    objdir = os.path.join(os.path.dirname(PKG_DIR), "build", ARCH + "_" + tag)
    os.makedirs(objdir, exist_ok=True)
    hdr_t = max([os.path.getmtime(h) for h in _headers()] + [0.0])

    def compile_one(src):
        obj = os.path.join(objdir, os.path.basename(src) + ".o")
        if not force and os.path.exists(obj) and os.path.getmtime(obj) > max(os.path.getmtime(src), hdr_t):
            return obj
        cmd = [hipcc, f"--offload-arch={ARCH}", *FLAGS, *defs, "-I", CSRC, "-I", INCLUDE, "-c", src, "-o", obj + ".tmp"]
        if verbose:
            print("[itts build]", os.path.basename(src), " ".join(defs), flush=True)
        subprocess.run(cmd, check=True)
        kernel = CHECKED.get(os.path.basename(src))
        if kernel:
            subprocess.run([*cmd[:cmd.index("-c")], "--cuda-device-only", "-S", src, "-o", obj + ".s"], check=True)
            with open(obj + ".s") as f:
                if not check_products(f.read(), kernel):
                    raise RuntimeError(f"no products of {kernel} in the assembly of {src}")
        os.replace(obj + ".tmp", obj)
        return obj

    jobs = max(1, min(len(sources()), int(os.environ.get("MAX_JOBS", os.cpu_count() or 4)), 16))
    with ThreadPoolExecutor(jobs) as ex:
        objs = list(ex.map(compile_one, sources()))
    tmp = out + ".tmp"
    subprocess.run([hipcc, f"--offload-arch={ARCH}", "-shared", "-fPIC", "-o", tmp, *objs], check=True)
    os.replace(tmp, out)
    if verbose:
        print("[itts build] linked", out, flush=True)
    return out


if __name__ == "__main__":
    build(force="--force" in sys.argv)
