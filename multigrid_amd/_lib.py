"""ctypes binding of ``libmgrid_hip.so`` (declared in ``include/mgrid.h``).

There is no CPU fallback: if the HIP library has not been built, importing a symbol
from here raises, and every product path stops with it.
"""
from __future__ import annotations

import ctypes
import os
import subprocess

PKG_DIR = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(PKG_DIR)
LIB_PATH = os.environ.get("MGRID_LIB", os.path.join(PKG_DIR, "libmgrid_hip.so"))
SRC_PATH = os.path.join(PKG_DIR, "csrc", "mgrid.hip")
POLICY_PATH = os.path.join(PKG_DIR, "csrc", "policy.hip")
TORCH_SRC_PATH = os.path.join(PKG_DIR, "csrc", "policy_torch.cpp")
TORCH_LIB_PATH = os.path.join(PKG_DIR, "_policy_torch.so")
INCLUDE_DIR = os.path.join(ROOT, "include")

MG_OK = 0
KIND_EMPTY, KIND_REDBLUEDOORS, KIND_BLOCKEDUNLOCKPICKUP, KIND_LOCKEDHALLWAY, KIND_COMPETITIVE = range(5)
AUTORESET_NONE, AUTORESET_SAME_STEP, AUTORESET_NEXT_STEP = range(3)
NUM_STATS = 8
ABI_VERSION = 9
ONE_HOT_DIM = 24  # 11 types + 6 colours + 7 states, multigrid/wrappers.py:95

EXPORTS = ("mg_abi_version", "mg_create", "mg_destroy", "mg_last_error", "mg_upload_layouts", "mg_generate_layouts",
           "mg_set_reward_schemes",
           "mg_reset", "mg_step", "mg_step_shards", "mg_step_n", "mg_gen_obs", "mg_gen_obs_of_state", "mg_get_state", "mg_set_state",
           "mg_stats", "mg_episode_stats", "mg_agents_mask", "mg_launch_census",
           "mg_embed", "mg_embed_grad_workspace", "mg_embed_grad", "mg_adjust_logits", "mg_adjust_logits_grad",
           "mg_draw_workspace", "mg_draw", "mg_token_logprobs_workspace", "mg_token_logprobs", "mg_token_logprobs_grad")
# element types, types of ids and tokens, kinds of masks (include/mgrid.h)
F32, BF16, F16, F64 = range(4)
U8, I32, I64 = range(3)
MASK_NONE, MASK_BYTES, MASK_BITS = range(3)
MAX_FIELDS = 8


class MgConfig(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in (
        "kind", "width", "height", "num_agents", "view_size", "max_steps", "see_through_walls",
        "allow_agent_overlap", "joint_reward", "success_any", "failure_any", "num_rooms",
        "num_envs", "device", "autoreset", "env_id_offset", "death_match", "per_agent_outputs")] + [
        ("seed", ctypes.c_uint64), ("batch_envs", ctypes.c_int32), ("reserved0", ctypes.c_int32)]


class MgOut(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in (
        "image_dev", "direction_dev", "reward_dev", "terminated_dev", "truncated_dev", "onehot_dev",
        "rows_dev", "reward64_dev", "info_dev")]


class MgLayoutSpec(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int32) for n in (
        "size", "random_start", "start_x", "start_y", "start_dir", "max_hallway_keys",
        "max_keys_per_room")] + [("agent_color", ctypes.c_uint8 * 64)]


class MgEmbed(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int64)] + [(n, ctypes.c_int32) for n in ("fields", "dim", "ids_type", "dtype")] + [
        (n, ctypes.c_int64) for n in ("ids_stride", "field_stride", "row_stride")] + [
        ("sizes", ctypes.c_int32 * MAX_FIELDS), ("scale", ctypes.c_float), ("reserved0", ctypes.c_int32), ("ids_copy_dev", ctypes.c_void_p)]


class MgAdjust(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int64), ("k", ctypes.c_int32), ("dtype", ctypes.c_int32)] + [
        (n, ctypes.c_int64) for n in ("logits_stride", "out_stride", "grad_stride")] + [
        ("history_dev", ctypes.c_void_p), ("lengths_dev", ctypes.c_void_p), ("history_stride", ctypes.c_int64),
        ("history_type", ctypes.c_int32), ("t", ctypes.c_int32)] + [
        (n, ctypes.c_void_p) for n in ("repetition_dev", "presence_dev", "frequency_dev")] + [
        (n, ctypes.c_float) for n in ("repetition", "presence", "frequency")] + [
        ("mask_kind", ctypes.c_int32), ("bias_dev", ctypes.c_void_p), ("bias_stride", ctypes.c_int64),
        ("mask_dev", ctypes.c_void_p), ("mask_stride", ctypes.c_int64)]


class MgLogits(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int64), ("k", ctypes.c_int32), ("dtype", ctypes.c_int32), ("stride", ctypes.c_int64),
                ("temperature_dev", ctypes.c_void_p), ("temperature", ctypes.c_float), ("tokens_type", ctypes.c_int32)]


def kernel_resources(listing: str):
    """Registers and spills of every kernel in a device assembly listing (the `amdhsa.kernels` metadata hipcc
    writes at its end): ``{mangled name: {vgpr_count, agpr_count, sgpr_count, sgpr_spill_count, vgpr_spill_count,
    private_segment_fixed_size, group_segment_fixed_size}}``."""
    import re
    text = open(listing).read()
    at = text.find("amdhsa.kernels:")
    out = {}
    if at < 0:
        return out
    for entry in re.split(r"\n  - ", text[at:])[1:]:
        name = re.search(r"\.name:\s+(\S+)", entry)
        if not name:
            continue
        rec = {}
        for key in ("vgpr_count", "agpr_count", "sgpr_count", "sgpr_spill_count", "vgpr_spill_count",
                    "private_segment_fixed_size", "group_segment_fixed_size"):
            m = re.search(r"\.%s:\s+(\d+)" % key, entry)
            rec[key] = int(m.group(1)) if m else 0
        out[name.group(1)] = rec
    return out


def _demangle(names):
    import shutil
    tool = shutil.which("c++filt") or shutil.which("llvm-cxxfilt", path="/opt/rocm/lib/llvm/bin")
    if not tool:
        return list(names)
    r = subprocess.run([tool], input="\n".join(names), capture_output=True, text=True)
    got = r.stdout.split("\n")[:len(names)]
    return got if r.returncode == 0 and len(got) == len(names) else list(names)


REGISTERS_PATH = os.path.join(PKG_DIR, "kernel_registers.json")


def torch_command(out: str):
    """The host compiler's line for the torch side of the policy operators, a Python extension module."""
    import sysconfig
    from torch.utils import cpp_extension
    include = [*cpp_extension.include_paths(), sysconfig.get_paths()["include"], "/opt/rocm/include", INCLUDE_DIR]
    return [os.environ.get("CXX", "g++"), "-O2", "-std=c++17", "-fPIC", "-shared", "-fvisibility=hidden", "-D__HIP_PLATFORM_AMD__=1", "-DUSE_ROCM=1",
            "-DTORCH_EXTENSION_NAME=_policy_torch", *(f"-I{p}" for p in include), TORCH_SRC_PATH, "-o", out,
            *(f"-L{p}" for p in cpp_extension.library_paths()), "-lc10", "-ltorch", "-ltorch_cpu", "-ltorch_python", "-lc10_hip"]


def build(force: bool = False, verbose: bool = False, extra_flags=(), out_path: str | None = None) -> str:
    """Compile the HIP library for gfx950 in-tree (hipcc cross-compiles without a GPU).

    The build keeps its intermediate files in a scratch directory and looks at the device assembly before the
    library is put in place: every kernel's register and spill counts are listed (``kernel_registers.json`` beside
    the library; printed with ``verbose``), a step or policy kernel that spills vector registers to scratch memory fails
    the build, and so does a code pattern this compiler was seen to get wrong (see _isa_lint.py)."""
    target = out_path or LIB_PATH
    sources = [SRC_PATH, POLICY_PATH, os.path.join(PKG_DIR, "csrc", "mgrid_experiment.h"),
               os.path.join(PKG_DIR, "csrc", "mgrid_error.h"), os.path.join(INCLUDE_DIR, "mgrid.h")]
    newest = max(os.path.getmtime(f) for f in sources)
    with_torch = out_path is None  # (a tuning build elsewhere is the HIP library alone)
    made = {target: newest}
    if with_torch:
        made[TORCH_LIB_PATH] = max(os.path.getmtime(f) for f in (TORCH_SRC_PATH, os.path.join(INCLUDE_DIR, "mgrid.h")))
    if not force and all(os.path.exists(f) and os.path.getmtime(f) >= t for f, t in made.items()):
        return target
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    # mgrid.hip at -Os, measured: the step kernel is 7 % faster than at -O3 (smaller code, and 126 instead of 129
    # vector registers, which lets a fourth wavefront onto every SIMD).  The streaming kernels of policy.hip are unrolled
    # where it pays: -O2.  Packed float32 instructions (v_pk_add_f32 and its like) are to stay out of the device code,
    # some of their forms have given wrong results: policy.hip is compiled without them; in mgrid.hip the compiler finds
    # no use for them, while the switch itself costs nine of its kernels two spilled registers each.  The listings of
    # both are searched for them below.
    no_packed = ("-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops")
    import glob
    import json
    import re
    import shutil
    import tempfile
    from ._isa_lint import find_masked_copies
    tmp = tempfile.mkdtemp(prefix="mgrid_build_")
    running = []
    try:
        out = os.path.join(tmp, "libmgrid_hip.so")
        objects = []
        for path, level in ((SRC_PATH, ("-Os",)), (POLICY_PATH, ("-O2", *no_packed))):  # side by side
            objects.append(os.path.join(tmp, os.path.basename(path) + ".o"))
            cmd = [hipcc, *level, "-std=c++17", "--offload-arch=gfx950", "-fPIC", "-c", "-save-temps", "-I", INCLUDE_DIR,
                   *extra_flags, path, "-o", objects[-1]]
            if verbose:
                print(" ".join(cmd))
            running.append((cmd, subprocess.Popen(cmd, cwd=tmp)))
        torch_out = os.path.join(tmp, "_policy_torch.so")
        if with_torch:
            cmd = torch_command(torch_out)
            if verbose:
                print(" ".join(cmd))
            running.append((cmd, subprocess.Popen(cmd, cwd=tmp)))
        for cmd, process in running:
            if process.wait() != 0:
                raise subprocess.CalledProcessError(process.returncode, cmd)
        subprocess.check_call([hipcc, "--offload-arch=gfx950", "-fPIC", "-shared", *objects, "-o", out], cwd=tmp)
        listings = glob.glob(os.path.join(tmp, "*gfx950*.s"))
        if not listings:
            raise RuntimeError("the build left no device assembly to check")
        report, spilling = {}, []
        for path in listings:
            hits = find_masked_copies(path)
            if hits:
                what = "; ".join(f"{k} {label}: {ins[0]}" for k, label, ins in hits[:3])
                raise RuntimeError(f"device code writes vector registers before a divergent region's lanes are "
                                   f"switched back on ({len(hits)} place(s): {what}); change the source around the "
                                   "named kernel until the compiler stops doing that")
            packed = re.search(r"\bv_pk_(add|mul|fma)_f32\b", open(path).read())
            if packed:
                raise RuntimeError(f"{os.path.basename(path)} holds {packed.group(0)}")
            res = kernel_resources(path)
            for mangled, plain in zip(res, _demangle(list(res))):
                name = plain.replace("(anonymous namespace)::", "")
                report[name] = res[mangled]  # template arguments of mg_tile_kernel: view, see-through, MODE (0 = step), ...
                # (a private segment without spilled vector registers is a frame object the compiler reserved and then
                # never touched - the listing has no scratch instruction for it; it is reported, not refused)
                if res[mangled]["vgpr_spill_count"] and ("mg_tile_kernel" in name or "policy" in os.path.basename(path)):
                    spilling.append((name, res[mangled]))
        if verbose:
            for k in sorted(report):
                r = report[k]
                print(f"  {r['vgpr_count']:3d} vgpr {r['sgpr_count']:3d} sgpr  spills {r['sgpr_spill_count']:3d} s / "
                      f"{r['vgpr_spill_count']:3d} v  scratch {r['private_segment_fixed_size']:4d} B  {k}")
        if spilling and os.environ.get("MGRID_ALLOW_SPILLS") != "1":  # (the switch is for work in progress only)
            raise RuntimeError(f"{len(spilling)} instantiation(s) of the tile or policy kernels spill vector registers to "
                               f"scratch memory, e.g. {spilling[0][0]}: {spilling[0][1]}")
        # a new inode, renamed into place: processes that have the old library mapped keep the old file
        for built, place in ((out, target), (torch_out, TORCH_LIB_PATH)) if with_torch else ((out, target),):
            staged = f"{place}.tmp.{os.getpid()}"
            shutil.copy2(built, staged)
            os.replace(staged, place)
        if out_path is None:
            with open(REGISTERS_PATH, "w") as f:
                json.dump(report, f, indent=1, sort_keys=True)
                f.write("\n")
    finally:
        for _, process in running:
            if process.poll() is None:
                process.kill()
            process.wait()
        shutil.rmtree(tmp, ignore_errors=True)
    return target


_lib = None


def lib() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; "
                "g.build()'` (there is no CPU fallback for the MI355X path)")
        L = ctypes.CDLL(LIB_PATH)
        vp, i32 = ctypes.c_void_p, ctypes.c_int32
        L.mg_abi_version.restype = ctypes.c_int
        L.mg_create.argtypes = [ctypes.POINTER(MgConfig), ctypes.POINTER(vp)]
        L.mg_destroy.argtypes = [vp]
        L.mg_last_error.argtypes = [vp]
        L.mg_last_error.restype = ctypes.c_char_p
        L.mg_upload_layouts.argtypes = [vp, vp, vp, vp, i32]
        if hasattr(L, "mg_set_reward_schemes"):  # (tuning builds of older sources loaded through MGRID_LIB lack it)
            L.mg_set_reward_schemes.argtypes = [vp, vp]
        L.mg_generate_layouts.argtypes = [vp, ctypes.POINTER(MgLayoutSpec), i32, ctypes.c_uint64]
        L.mg_reset.argtypes = [vp, vp, vp, ctypes.POINTER(MgOut), vp]
        L.mg_step.argtypes = [vp, vp, vp, ctypes.POINTER(MgOut), vp]
        if hasattr(L, "mg_step_shards"):
            L.mg_step_shards.argtypes = [ctypes.POINTER(vp), i32, vp, vp, ctypes.POINTER(MgOut), ctypes.POINTER(vp)]
        L.mg_step_n.argtypes = [vp, i32, vp, vp, ctypes.POINTER(MgOut), vp]
        L.mg_gen_obs.argtypes = [vp, ctypes.POINTER(MgOut), vp]
        L.mg_gen_obs_of_state.argtypes = [ctypes.POINTER(MgConfig), vp, vp, ctypes.POINTER(MgOut), vp]
        L.mg_get_state.argtypes = [vp] * 7
        L.mg_set_state.argtypes = [vp] * 7
        L.mg_stats.argtypes = [vp, vp, vp]
        if hasattr(L, "mg_agents_mask"):
            L.mg_agents_mask.argtypes = [vp, vp, vp, vp]
        if hasattr(L, "mg_episode_stats"):
            L.mg_episode_stats.argtypes = [i32, i32] + [vp] * 9
        if hasattr(L, "mg_launch_census"):
            L.mg_launch_census.argtypes = [ctypes.c_char_p, i32]
        if hasattr(L, "mg_embed"):
            i64, emb, adj, lgt = ctypes.c_int64, ctypes.POINTER(MgEmbed), ctypes.POINTER(MgAdjust), ctypes.POINTER(MgLogits)
            L.mg_embed.argtypes = [emb] + [vp] * 4
            L.mg_embed_grad.argtypes = [emb] + [vp] * 4 + [i64, vp]
            L.mg_adjust_logits.argtypes = [adj] + [vp] * 3
            L.mg_adjust_logits_grad.argtypes = [adj] + [vp] * 4
            L.mg_draw.argtypes = [lgt, vp, vp, i32] + [vp] * 3 + [i64, vp]
            L.mg_token_logprobs.argtypes = [lgt] + [vp] * 6 + [i64, vp]
            L.mg_token_logprobs_grad.argtypes = [lgt] + [vp] * 4 + [i64, vp, i64, vp, vp]
            for name, arg in (("mg_embed_grad_workspace", emb), ("mg_draw_workspace", lgt), ("mg_token_logprobs_workspace", lgt)):
                getattr(L, name).argtypes = [arg]
        for name in EXPORTS:
            if name.endswith("_workspace") and hasattr(L, name):
                getattr(L, name).restype = ctypes.c_int64
            elif name not in ("mg_last_error",) and hasattr(L, name):
                getattr(L, name).restype = ctypes.c_int
        _lib = L
    return _lib


def launch_census() -> dict:
    """``{(V, SEE, MODE, WALLED, OH, MULTI, COMP, CROWD, STG): launches}`` of this process so far (``mg_launch_census``)."""
    buf = ctypes.create_string_buffer(1 << 16)
    check(lib().mg_launch_census(buf, len(buf)))
    out = {}
    for line in buf.value.decode().splitlines():
        what, n = line.split(":")
        out[tuple(int(x) for x in what.split(","))] = int(n)
    return out


def compiled_instantiations() -> set:
    """The instantiations of the tile kernel the library was built with, from the build's register report
    (``kernel_registers.json``), as tuples like the keys of ``launch_census``."""
    import json
    import re
    out = set()
    for name in json.load(open(REGISTERS_PATH)):
        m = re.search(r"mg_tile_kernel<([^>]*)>", name)
        if m:
            out.add(tuple({"true": 1, "false": 0}.get(x.strip(), None) if x.strip() in ("true", "false") else int(x)
                          for x in m.group(1).split(",")))
    return out


class MgError(RuntimeError):
    pass


def check(rc: int, handle=None):
    if rc != MG_OK:
        msg = lib().mg_last_error(handle)
        raise MgError(f"libmgrid_hip error {rc}: {msg.decode() if msg else '?'}")
