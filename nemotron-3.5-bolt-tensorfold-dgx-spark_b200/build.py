"""Build libb200q.so in place: every csrc/*.cu compiled by nvcc for sm_100a (-gencode arch=compute_100a,code=sm_100a)
and linked into one shared library beside this file.

The ggml IQ2_XXS tables are compiled in from the reference's own table file, found by path (B200Q_IQ2_TABLES, else
engine/iq2_tables.inc of a reference checkout named "reference" beside this repository); they are not copied into the
sources.  Where that file is absent (a machine that only runs), the prebuilt library is used, and only if it was built from these
sources: a stale prebuilt library is an error, never reused and never replaced by less.  With neither, the sources that do not
need the tables (TABLE_FREE) are built into a library of another name, PART: calling an operator that it lacks raises.
"""
import concurrent.futures
import hashlib
import os
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(HERE)
CSRC = os.path.join(HERE, "csrc")
OUT = os.path.join(HERE, "libb200q.so")
PART = os.path.join(HERE, "libb200q_tablefree.so")   # b200q.py loads it where OUT is missing
OBJ = os.path.join(HERE, "_build")
TABLES = os.environ.get("B200Q_IQ2_TABLES",
                        os.path.join(os.path.dirname(ROOT), "reference", "engine", "iq2_tables.inc"))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
ARCH = ["-gencode", "arch=compute_100a,code=sm_100a"]
FLAGS = ["-O3", "-std=c++17", "-lineinfo", "-Xcompiler", "-fPIC", "--expt-relaxed-constexpr",
         "-Xptxas", "-warn-spills", f"-DB200Q_IQ2_TABLES=\"{TABLES}\"", "-I", os.path.join(ROOT, "include")]


# the sources that neither read the IQ2_XXS tables nor call code that does
TABLE_FREE = ("attn_decode.cu", "attn_prompt.cu", "core.cu", "gemv_tc.cu", "kv.cu", "nv4_gemm.cu")


def sources():
    return sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith(".cu"))


def _all_sources():
    inc = os.path.join(ROOT, "include")
    return (sources() + [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith((".cuh", ".h"))] +
            [os.path.join(inc, h) for h in os.listdir(inc) if h.endswith(".h")])


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


def _compile(src, verbose=False):
    obj = os.path.join(OBJ, os.path.basename(src)[:-3] + ".o")
    headers = [os.path.join(CSRC, h) for h in os.listdir(CSRC) if h.endswith((".cuh", ".h"))]
    inc = os.path.join(ROOT, "include")
    headers += [os.path.join(inc, h) for h in os.listdir(inc) if h.endswith(".h")]
    if not _stale(obj, [src, __file__] + headers):
        return obj
    cmd = [NVCC, *ARCH, *FLAGS, "-c", src, "-o", obj]
    if verbose:
        cmd.insert(1, "-Xptxas=-v")
    r = subprocess.run(cmd, capture_output=True, text=True)
    if r.returncode != 0:
        raise RuntimeError(f"nvcc failed on {src}:\n{r.stderr}")
    if verbose and r.stderr:
        sys.stderr.write(r.stderr)
    return obj


def _digest():
    h = hashlib.sha256()
    for f in sorted(_all_sources()):
        with open(f, "rb") as src:
            h.update(os.path.basename(f).encode() + b"\0" + hashlib.sha256(src.read()).digest())
    return h.hexdigest()


def _record(out):
    """what `out` was linked from, as written beside it: [digest of the sources, objects ..]; [] if nothing says"""
    try:
        with open(out + ".sources") as f:
            return f.read().split()
    except FileNotFoundError:
        return []


def _prebuilt_is_current():
    """by the sources' contents, or by their times where nothing is recorded: times change when a tree is copied"""
    record = _record(OUT)
    return record[0] == _digest() if record else not _stale(OUT, _all_sources())


def build(force=False, verbose=False):
    """Compile and link libb200q.so (without the tables and a prebuilt one: PART); returns the library's path."""
    srcs, out = sources(), OUT
    if not os.path.exists(TABLES):
        if os.path.exists(OUT):
            if _prebuilt_is_current():
                return OUT
            raise RuntimeError(f"IQ2_XXS table file not found at {TABLES}, and the prebuilt {OUT} is not of these sources")
        sys.stderr.write(f"IQ2_XXS table file not found at {TABLES}: {os.path.basename(PART)} lacks the operators that need it\n")
        srcs, out = [s for s in srcs if os.path.basename(s) in TABLE_FREE], PART
    os.makedirs(OBJ, exist_ok=True)
    if force:
        for f in os.listdir(OBJ):
            os.remove(os.path.join(OBJ, f))
    with concurrent.futures.ThreadPoolExecutor(max_workers=min(8, len(srcs))) as ex:
        objs = list(ex.map(lambda s: _compile(s, verbose), srcs))
    names = [os.path.basename(o) for o in objs]
    if force or _stale(out, objs) or _record(out)[1:] != names:
        cmd = [NVCC, *ARCH, "-shared", "-o", out, *objs, "-lcuda"]
        r = subprocess.run(cmd, capture_output=True, text=True)
        if r.returncode != 0:
            raise RuntimeError(f"link failed:\n{r.stderr}")
    record = [_digest(), *names]
    if _record(out) != record:
        with open(out + ".sources", "w") as f:
            f.write("\n".join(record) + "\n")
    return out


if __name__ == "__main__":
    print(build(force="--force" in sys.argv, verbose="-v" in sys.argv))
