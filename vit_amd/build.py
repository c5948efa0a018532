"""Build libvitk.so (the HIP kernels + C ABI) in-tree with plain hipcc.

    python -m vit_amd.build [--force]

No torch headers are involved: the library is a bare `hipcc -shared -fPIC
--offload-arch=gfx950` product, loaded with ctypes (vit_amd/lib.py).  hipcc
cross-compiles gfx950 code without a GPU.
"""
import os
import re
import subprocess
import sys
from concurrent.futures import ThreadPoolExecutor

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIB = os.path.join(HERE, "libvitk.so")
SOURCES = ["vitk_api.hip", "gemm.hip", "gemm_pipe.hip", "gemm_pp.hip", "attention.hip", "rowops.hip", "f32path.hip", "backward.hip", "gemm_tn.hip", "attention_bwd.hip",
           "group_norm.hip", "grad_clip.hip", "diff_attention.hip", "diff_attention_bwd.hip"]
HEADERS = [os.path.join(CSRC, "vitk_common.h"), os.path.join(CSRC, "vitk_kernels.h"), os.path.join(CSRC, "gemm_common.h"), os.path.join(CSRC, "gemm_plan.h"), os.path.join(CSRC, "diff_attention.h"),
           os.path.join(os.path.dirname(HERE), "include", "vitk.h")]
# Packed f32 instructions (v_pk_add/mul/fma_f32) are switched off: some of their forms have given wrong results on this
# hardware now and then, without an error, and -O3 makes them from ordinary float code by itself.
FLAGS = ["-O3", "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-ffp-contract=fast",
         "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]


def _hipcc():
    for c in (os.environ.get("HIPCC"), "/opt/rocm/bin/hipcc", "hipcc"):
        if c and (os.path.isabs(c) and os.path.exists(c) or not os.path.isabs(c)):
            return c
    return "hipcc"


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def build(force=False, verbose=True, probes=False):
    """Compile every .hip source to an object (in parallel) and link libvitk.so.  probes=True builds the
    diagnostic library libvitk_probes.so instead (-DVITK_PROBES: timing probes that give wrong or no results,
    for tools/ only; select it with VITK_LIB=...)."""
    objdir = os.path.join(HERE, "build_probes" if probes else "build")
    lib = os.path.join(HERE, "libvitk_probes.so") if probes else LIB
    os.makedirs(objdir, exist_ok=True)
    hipcc = _hipcc()
    jobs = []
    for src in SOURCES:
        s = os.path.join(CSRC, src)
        o = os.path.join(objdir, src.replace(".hip", ".o"))
        if force or _stale(o, [s, __file__] + HEADERS):
            jobs.append((s, o))

    def compile_one(job):
        s, o = job
        cmd = [hipcc] + FLAGS + (["-DVITK_PROBES"] if probes else []) + ["-c", s, "-o", o]
        if verbose:
            print("[vit_amd.build]", " ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)

    if jobs:
        with ThreadPoolExecutor(max_workers=min(4, len(jobs))) as ex:
            list(ex.map(compile_one, jobs))
    objs = [os.path.join(objdir, s.replace(".hip", ".o")) for s in SOURCES]
    if force or jobs or _stale(lib, objs):
        cmd = [hipcc, "-shared", "-fPIC", "--offload-arch=gfx950", "-o", lib] + objs
        if verbose:
            print("[vit_amd.build]", " ".join(cmd), flush=True)
        subprocess.run(cmd, check=True)
    return lib


# Sources whose transposed LDS reads are looked at in the compiled code.  gemm_tn.hip waits for inline-asm LDS reads with
# counted `s_waitcnt lgkmcnt(n)`: the counts hold only while nothing else of the wave is outstanding on that counter.  LDS
# returns in order, scalar memory does not, so one scalar load (a kernel-argument or descriptor reload) between a
# transposed LDS read and the wait that covers it could let the wait pass early.  And the compiler does not know that such
# a read's result is still on its way, so it may copy or spill the register before the wait: that too fails the build.
# attention.hip leaves the waits of its reads to the compiler; its LDS-DMA is inline asm that the compiler does not know
# of, so a barrier that one reaches without the kernel's own wait fails the build.
COUNTED_WAIT_SOURCES = ["attention.hip", "gemm_tn.hip"]


def scan_counted_waits(asm_text):
    """(kernel, line number, instruction) of every scalar-memory instruction that sits, in program text order, between
    a ds_read_b64_tr_b16 and the next `s_waitcnt` with lgkmcnt(0) of the same kernel."""
    found, kernel, pending = [], None, False
    for ln, line in enumerate(asm_text.splitlines(), 1):
        t = line.strip()
        if re.match(r"^_Z\w+:", t):
            kernel, pending = t[:-1], False
            continue
        if not t or t[0] in ";.":
            continue
        ins = t.split()[0]
        if ins == "ds_read_b64_tr_b16":
            pending = True
        elif ins == "s_waitcnt":
            m = re.search(r"lgkmcnt\((\d+)\)", t)
            if m and int(m.group(1)) == 0:
                pending = False
        elif pending and ins.startswith(("s_load_", "s_buffer_load_", "s_memtime", "s_memrealtime", "s_dcache")):
            found.append((kernel, ln, t))
    return found


def _asm_kernels(asm_text):
    """(name, [(line number, instruction or label)]) of every function in compiler-written assembly."""
    name, body = None, []
    for ln, line in enumerate(asm_text.splitlines(), 1):
        t = line.split(";")[0].strip()
        if re.match(r"^_Z\w+:", t):
            name, body = t[:-1], []
        elif name and t.startswith(".Lfunc_end"):
            yield name, body
            name = None
        elif name and t and (t[0] != "." or t.endswith(":")):
            body.append((ln, t))
    if name:
        yield name, body


def _vector_registers(operands):
    regs = set()
    for one, lo, hi in re.findall(r"\bv(?:(\d+)|\[(\d+):(\d+)\])", operands):
        regs.update([int(one)] if one else range(int(lo), int(hi) + 1))
    return regs


def scan_in_flight(asm_text):
    """(kernel, line number, instruction) of every instruction that touches the result of a transposed LDS read before a
    wait that covers the read, and of every barrier that an LDS-DMA reaches without an `s_waitcnt` with vmcnt(0), along any
    path through a kernel.  A read is covered by lgkmcnt(n) if n LDS instructions or more have followed it, since LDS
    returns in order."""
    found = []
    for kernel, body in _asm_kernels(asm_text):
        blocks, label = [[]], {}
        for ln, t in body:
            if t.endswith(":"):
                blocks.append([])
                label[t[:-1]] = len(blocks) - 1
                continue
            blocks[-1].append((ln, t))
            if t.startswith(("s_branch", "s_cbranch", "s_endpgm")):
                blocks.append([])
        after = [[i + 1] if i + 1 < len(blocks) else [] for i in range(len(blocks))]
        for i, b in enumerate(blocks):
            op = b[-1][1].split() if b else [""]
            if op[0] in ("s_branch", "s_endpgm"):
                after[i] = []
            if op[0].startswith(("s_branch", "s_cbranch")):
                after[i] = after[i] + [label[op[1]]]
        # state: in-flight register -> LDS instructions since its read (the fewest over all paths), "dma" -> 0 if one is out
        states, work, bad = {0: {}}, [0], {}
        while work:
            i = work.pop()
            st = dict(states[i])
            for ln, t in blocks[i]:
                op, _, rest = t.partition(" ")
                if op == "s_waitcnt":
                    m = re.search(r"lgkmcnt\((\d+)\)", t)
                    if m:
                        st = {r: n for r, n in st.items() if r == "dma" or n < int(m.group(1))}
                    if "vmcnt(0)" in t:
                        st.pop("dma", None)
                    continue
                is_read = op == "ds_read_b64_tr_b16"
                dst, _, src = rest.partition(",") if is_read else ("", "", rest)
                if _vector_registers(src) & st.keys() or op == "s_barrier" and "dma" in st:
                    bad[ln] = t
                if op.startswith("ds_"):
                    st = {r: n if r == "dma" else n + 1 for r, n in st.items()}
                for r in _vector_registers(dst):
                    st[r] = 0
                if "_lds_" in op and op.startswith(("global_load", "buffer_load")):
                    st["dma"] = 0
            for j in after[i]:
                old = states.get(j)
                new = dict(st) if old is None else {r: min(n for n in (old.get(r), st.get(r)) if n is not None) for r in old.keys() | st.keys()}
                if new != old:
                    states[j] = new
                    work.append(j)
        found += [(kernel, ln, t) for ln, t in sorted(bad.items())]
    return found


def scan_packed_f32(asm_text):
    """(kernel, line number, instruction) of every packed f32 instruction."""
    return [(k, ln, t) for k, body in _asm_kernels(asm_text) for ln, t in body if re.match(r"v_pk_(add|mul|fma)_f32\b", t)]


def check_counted_waits(verbose=True):
    """Compile COUNTED_WAIT_SOURCES to gfx950 assembly (cached beside the objects) and fail if the compiler put a
    scalar-memory instruction inside a counted-wait region, uses a transposed LDS read's result before its wait,
    or made packed f32 instructions."""
    objdir = os.path.join(HERE, "build")
    os.makedirs(objdir, exist_ok=True)
    hipcc = _hipcc()

    def asm_of(src):
        s, out = os.path.join(CSRC, src), os.path.join(objdir, src.replace(".hip", ".s"))
        if _stale(out, [s, __file__] + HEADERS):
            cmd = [hipcc] + FLAGS + ["-S", "--cuda-device-only", s, "-o", out]
            if verbose:
                print("[vit_amd.build]", " ".join(cmd), flush=True)
            subprocess.run(cmd, check=True, stderr=subprocess.DEVNULL)
        return out

    with ThreadPoolExecutor(max_workers=len(COUNTED_WAIT_SOURCES)) as ex:
        outs = list(ex.map(asm_of, COUNTED_WAIT_SOURCES))
    for src, out in zip(COUNTED_WAIT_SOURCES, outs):
        with open(out) as f:
            asm = f.read()
        bad = scan_counted_waits(asm)
        if bad:
            k, ln, ins = bad[0]
            raise RuntimeError(f"{src}: {len(bad)} scalar-memory instruction(s) inside a counted lgkmcnt wait region, "
                               f"first in {k} at {os.path.basename(out)}:{ln}: {ins}")
        bad = scan_in_flight(asm)
        if bad:
            k, ln, ins = bad[0]
            raise RuntimeError(f"{src}: {len(bad)} instruction(s) ahead of the wait for a transposed LDS read or an LDS-DMA, "
                               f"first in {k} at {os.path.basename(out)}:{ln}: {ins}")
        bad = scan_packed_f32(asm)
        if bad:
            k, ln, ins = bad[0]
            raise RuntimeError(f"{src}: {len(bad)} packed f32 instruction(s), first in {k} at {os.path.basename(out)}:{ln}: {ins}")
    return True


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, probes="--probes" in sys.argv))
    if "--check-waits" in sys.argv:
        print("counted waits clean:", check_counted_waits())
