"""Build libsoundbubble_hip.so (gfx950) in-tree with hipcc -- no torch dependency -- and, beside it, libsoundbubble_torch.so: the
sequence-block operators' calls from PyTorch (csrc/seq/sb_seq_torch.cpp), host code against the headers of the torch that is installed.
Without a torch, a host compiler or Python's headers the first is built alone; the operators then go through their Python wrappers."""
import os
import shutil
import subprocess
import sys

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(HERE, "csrc")
LIBDIR = os.path.join(HERE, "lib")
LIB = os.path.join(LIBDIR, "libsoundbubble_hip.so")
SOURCES = ["sb_lstm.hip", "sb_lstm_gen.hip", "sb_lstm_vec.hip", "sb_lstm_bf_fwd.hip", "sb_lstm_bf_bwd.hip", "sb_lstm_stream.hip", "sb_attention.hip",
           "sb_linear.hip", "sb_elementwise.hip", "sb_mrstft.hip"]
# the sequence-block operators (layer norm, gated linear recurrence, AdamW): a folder and a header of their own, so that the digest
# below stays the separator kernels'
SEQ_SOURCES = ["seq/sb_layer_norm.hip", "seq/sb_gated_scan.hip", "seq/sb_adamw.hip"]
HEADERS = [os.path.join(CSRC, "sb_common.h"), os.path.join(CSRC, "sb_lstm_bf_common.h"),
           os.path.join(HERE, "..", "include", "sound_bubble_hip.h")]
SEQ_HEADERS = [os.path.join(CSRC, "sb_common.h"), os.path.join(CSRC, "seq", "sb_seq_common.h"),
               os.path.join(HERE, "..", "include", "sound_bubble_seq.h")]


TORCH_LIB = os.path.join(LIBDIR, "libsoundbubble_torch.so")
TORCH_SOURCE = os.path.join(CSRC, "seq", "sb_seq_torch.cpp")


def torch_lib_cmd():
    """-> the compiler line of libsoundbubble_torch.so and a stamp, the line with the torch that it is for (which is looked up, not
    imported); None and the reason where there is nothing to build it with"""
    import importlib.util
    import sysconfig
    spec, cxx, include = importlib.util.find_spec("torch"), os.environ.get("CXX", "g++").split(), sysconfig.get_paths()["include"]
    t = spec.submodule_search_locations[0] if spec is not None else ""
    if not os.path.exists(os.path.join(t, "lib", "libc10_hip.so")):
        return None, "no torch for ROCm is installed"
    if shutil.which(cxx[0]) is None:
        return None, f"no {cxx[0]}"
    if not os.path.exists(os.path.join(include, "Python.h")):
        return None, "no Python.h"
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    cmd = [*cxx, "-O2", "-std=c++17", "-fPIC", "-shared", "-D__HIP_PLATFORM_AMD__", "-DUSE_ROCM", "-D_GLIBCXX_USE_CXX11_ABI=1",
           "-I" + os.path.join(t, "include"), "-I" + os.path.join(t, "include", "torch", "csrc", "api", "include"), "-I" + os.path.join(rocm, "include"),
           "-I" + include, TORCH_SOURCE, "-o", TORCH_LIB, "-L" + os.path.join(t, "lib"), "-lc10", "-lc10_hip", "-lamdhip64", "-ltorch_cpu", "-ltorch", "-ltorch_python"]
    with open(os.path.join(t, "version.py")) as f:
        return cmd, " ".join(cmd) + "\n" + f.read()


def _torch_job(force):
    """-> the compiler line of libsoundbubble_torch.so if it has to be built, and its stamp.  One that is stale and cannot be built is taken away: its
    calls' layout need not be the library's any more"""
    cmd, stamp = torch_lib_cmd()
    stale = force or _stale(TORCH_LIB, [TORCH_SOURCE, SEQ_HEADERS[-1]])
    if cmd is None:
        print(f"[build] libsoundbubble_torch.so is not built: {stamp}", flush=True)
        if stale and os.path.exists(TORCH_LIB):
            os.remove(TORCH_LIB)
        return None, ""
    if os.path.exists(TORCH_LIB + ".stamp"):
        with open(TORCH_LIB + ".stamp") as f:
            stale |= f.read() != stamp
    else:
        stale = True
    return (cmd if stale else None), stamp


def csrc_digest():
    """sha256 (first 16 hex digits) over the kernel sources and the C-ABI header, names and bytes in sorted order: what a
    committed counter profile is stamped with (scripts/pmc_summary.py) and what bench.py compares it against (`stale_profile`)"""
    import hashlib
    h = hashlib.sha256()
    files = sorted(os.path.join(CSRC, f) for f in os.listdir(CSRC) if f.endswith((".hip", ".h"))) + [os.path.normpath(HEADERS[-1])]
    for f in files:
        h.update(os.path.basename(f).encode())
        h.update(open(f, "rb").read())
    return h.hexdigest()[:16]


def _stale(target, deps):
    if not os.path.exists(target):
        return True
    t = os.path.getmtime(target)
    return any(os.path.getmtime(d) > t for d in deps)


# The recurrent kernels keep few accumulators: MFMA results straight into VGPRs saves the v_accvgpr_read copies (and
# their hazard nops) in front of every cell update (+2-3 % on the inference forward, training neutral; same-box A/B).
# The streaming / GEMM kernels hold ~100 accumulator registers and are better off with AGPRs (hipcc's default).
# -ffp-contract=off: every fused multiply-add in the recurrent kernels is written out (__builtin_fmaf), so all template
# variants of a kernel (e.g. the time-segmented and the plain schedule) round identically -- bit-exact outputs.
_BF_FLAGS = ["-mllvm", "-amdgpu-mfma-vgpr-form", "-ffp-contract=off"]
# no packed fp32 instructions in the sequence-block kernels: they wait for memory, and those forms are not needed for it; AdamW
# rounds every operation by itself (its 8-bit codes are defined by those roundings)
_SEQ_FLAGS = ["-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops"]
PER_FILE_FLAGS = {"sb_lstm_bf_fwd.hip": _BF_FLAGS, "sb_lstm_bf_bwd.hip": _BF_FLAGS,
                  "seq/sb_layer_norm.hip": _SEQ_FLAGS, "seq/sb_gated_scan.hip": _SEQ_FLAGS,
                  "seq/sb_adamw.hip": _SEQ_FLAGS + ["-ffp-contract=off"]}
# translation units built a second time with another macro set: (source, object stem, extra flags).  The opt-in two-product
# forward (sb_lstm_fwd_args.products == 2) is the forward file again with -DSB_FWD_2P: its inference kernels only, launcher
# sb_launch_lstm_fwd_bf_2p.
EXTRA_UNITS = [("sb_lstm_bf_fwd.hip", "sb_lstm_bf_fwd_2p", _BF_FLAGS + ["-DSB_FWD_2P"])]


def object_of(src):
    """the object of a source, or of the stem of one of EXTRA_UNITS"""
    return os.path.join(LIBDIR, os.path.basename(src).replace(".hip", "") + ".o")


def objects(instead=()):
    """what libsoundbubble_hip.so is linked from.  instead: {source or stem: another object} of an experiment's library, which has to
    export all that _lib.load() asks for"""
    return [dict(instead).get(u, object_of(u)) for u in SOURCES + SEQ_SOURCES + [stem for _, stem, _ in EXTRA_UNITS]]


def build(force=False, verbose=True):
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    os.makedirs(LIBDIR, exist_ok=True)
    objs, jobs = objects(), []
    for src in SOURCES + SEQ_SOURCES:
        s, o = os.path.join(CSRC, src), object_of(src)
        if force or _stale(o, [s] + (SEQ_HEADERS if src in SEQ_SOURCES else HEADERS)):
            cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-value", "-c", s, "-o", o]
            cmd[2:2] = os.environ.get("SB_EXTRA_HIPCC_FLAGS", "").split()     # e.g. -DSB_PHASE_TIMING (dev tool)
            cmd[2:2] = PER_FILE_FLAGS.get(src, [])
            jobs.append(cmd)
    for src, stem, flags in EXTRA_UNITS:
        s, o = os.path.join(CSRC, src), object_of(stem)
        if force or _stale(o, [s] + HEADERS):
            cmd = [hipcc, "--offload-arch=gfx950", "-O3", "-std=c++17", "-fPIC", "-Wno-unused-value", "-c", s, "-o", o]
            cmd[2:2] = os.environ.get("SB_EXTRA_HIPCC_FLAGS", "").split()
            cmd[2:2] = flags
            jobs.append(cmd)
    torch_job, stamp = _torch_job(force)

    def run(cmd):
        if verbose:
            print("[build]", " ".join(cmd), flush=True)
        subprocess.check_call(cmd)
    from concurrent.futures import ThreadPoolExecutor      # translation units are independent: compile them side by side
    with ThreadPoolExecutor(max_workers=max(1, min(len(jobs) + 1, (os.cpu_count() or 2) // 2))) as ex:
        beside = ex.submit(run, torch_job) if torch_job else None
        list(ex.map(run, jobs))
        if force or _stale(LIB, objs):
            run([hipcc, "--offload-arch=gfx950", "-shared", "-fPIC", "-o", LIB] + objs)
        if beside:
            beside.result()
            with open(TORCH_LIB + ".stamp", "w") as f:
                f.write(stamp)
    return LIB


if __name__ == "__main__":
    build(force="--force" in sys.argv)
