"""Python client of the C-ABI runner (libthrunner.so, include/thompiler_runner.h).

It mirrors the hackathon runner's two calls (the reference's docs/API.md):

  * ``compile_ptx(ptx)`` -> ``{"ok", "entry_points", "registers", "stage", "stderr", "module"}``
    (POST /compile; failures are returned with a stage, never raised);
  * ``run(...)`` on host numpy buffers -> ``{"ok", "median_us", "outputs", "stage", "stderr"}``
    (POST /run with args in arg_order, ``zero_outputs`` re-zeroed before
    every launch);

plus ``launch`` on device pointers for callers that keep data resident on
the GPU (PyTorch tensors), and the launch plan: meta.json's geometry, or the
tuned launch a family recorded in the PTX (``// @thompiler-launch``), with
the module globals (tensor maps, scratch words) that launch needs.

There is no fallback: without the built library every call raises.
"""

from __future__ import annotations

import ctypes
import operator
import re
import struct
from dataclasses import dataclass, field
from pathlib import Path

import numpy as np

from thompiler.emitter import read_sidecar

LIB_PATH = Path(__file__).resolve().parent.parent / "libthrunner.so"

STAGES = {1: "ptxas", 2: "lookup", 3: "run", 4: "request", 5: "timeout", 6: "cuda"}


class RunnerError(RuntimeError):
    def __init__(self, stage: str, message: str):
        super().__init__(f"[{stage}] {message}")
        self.stage = stage
        self.message = message


class ThrArg(ctypes.Structure):
    _fields_ = [("host", ctypes.c_void_p), ("nbytes", ctypes.c_uint64),
                ("kind", ctypes.c_int32), ("zero_each", ctypes.c_int32)]


class ThrTmapSpec(ctypes.Structure):
    _fields_ = [("global_", ctypes.c_char_p), ("arg", ctypes.c_int32), ("dtype_code", ctypes.c_int32),
                ("rank", ctypes.c_int32), ("swizzle", ctypes.c_int32), ("dims", ctypes.c_uint64 * 5),
                ("strides", ctypes.c_uint64 * 4), ("box", ctypes.c_uint32 * 5)]


class ThrRunDesc(ctypes.Structure):
    _fields_ = [("module", ctypes.c_uint64), ("function", ctypes.c_uint64), ("grid", ctypes.c_uint32 * 3),
                ("block", ctypes.c_uint32 * 3), ("smem_bytes", ctypes.c_uint32), ("nargs", ctypes.c_int32),
                ("args", ctypes.POINTER(ThrArg)), ("tmaps", ctypes.POINTER(ThrTmapSpec)), ("ntmaps", ctypes.c_int32),
                ("ptr_table", ctypes.c_char_p)]


class ThrLaunchDesc(ctypes.Structure):
    _fields_ = [("module", ctypes.c_uint64), ("function", ctypes.c_uint64), ("grid", ctypes.c_uint32 * 3),
                ("block", ctypes.c_uint32 * 3), ("smem_bytes", ctypes.c_uint32), ("flags", ctypes.c_uint32),
                ("nargs", ctypes.c_int32), ("ntmaps", ctypes.c_int32), ("align", ctypes.POINTER(ctypes.c_uint32)),
                ("tmaps", ctypes.POINTER(ThrTmapSpec)), ("ptr_table", ctypes.c_char_p)]


_lib = None


def library() -> ctypes.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RunnerError("cuda", f"runner library {LIB_PATH} is not built (run __graft_entry__.build())")
        lib = ctypes.CDLL(str(LIB_PATH))
        u64, i32, p = ctypes.c_uint64, ctypes.c_int, ctypes.c_void_p
        u32x3 = ctypes.POINTER(ctypes.c_uint32)
        sig = {
            "thr_version": ([], i32),
            "thr_init": ([i32], i32),
            "thr_device_info": ([i32, ctypes.POINTER(i32), ctypes.POINTER(i32), ctypes.POINTER(i32),
                                 ctypes.c_char_p, ctypes.c_size_t], i32),
            "thr_module_load": ([ctypes.c_char_p, ctypes.POINTER(u64), ctypes.c_char_p, ctypes.c_size_t], i32),
            "thr_module_unload": ([u64], i32),
            "thr_get_function": ([u64, ctypes.c_char_p, ctypes.POINTER(u64)], i32),
            "thr_function_attrs": ([u64] + [ctypes.POINTER(i32)] * 4, i32),
            "thr_module_global": ([u64, ctypes.c_char_p, ctypes.POINTER(u64), ctypes.POINTER(u64)], i32),
            "thr_launch": ([u64, u32x3, u32x3, ctypes.c_uint32, ctypes.POINTER(u64), i32, u64], i32),
            "thr_launch_ex": ([u64, u32x3, u32x3, ctypes.c_uint32, ctypes.POINTER(u64), i32, u64, ctypes.c_uint32],
                              i32),
            "thr_run": ([u64, u32x3, u32x3, ctypes.c_uint32, ctypes.POINTER(ThrArg), i32, i32, i32,
                         ctypes.c_double, ctypes.POINTER(ctypes.c_float), u64], i32),
            "thr_tensor_map": ([p, i32, i32, u64, ctypes.POINTER(u64), ctypes.POINTER(u64),
                                ctypes.POINTER(ctypes.c_uint32), i32], i32),
            "thr_run_ex": ([u64, u64, u32x3, u32x3, ctypes.c_uint32, ctypes.POINTER(ThrArg), i32,
                            ctypes.POINTER(ThrTmapSpec), i32, ctypes.c_char_p, i32, i32, ctypes.c_double,
                            ctypes.POINTER(ctypes.c_float), u64], i32),
            "thr_memcpy_htod": ([u64, p, u64, u64], i32),
            "thr_memcpy_dtoh": ([p, u64, u64], i32),
            "thr_synchronize": ([], i32),
            "thr_release_buffers": ([], i32),
            "thr_last_error": ([ctypes.c_char_p, ctypes.c_size_t], i32),
            "thr_run_batch": ([ctypes.POINTER(ThrRunDesc), i32, ctypes.c_double], i32),
            "thr_tmap_bind": ([u64, ctypes.POINTER(ThrTmapSpec), i32, ctypes.c_char_p, ctypes.POINTER(u64), i32,
                               u64, ctypes.POINTER(i32)], i32),
            "thr_tmap_launched": ([u64, i32, u64], i32),
            "thr_launch_prepared": ([p, ctypes.c_char_p, u64], i32),
            "thr_peer_alloc": ([u64, ctypes.POINTER(u64), ctypes.c_char_p], i32),
            "thr_peer_open": ([ctypes.c_char_p, ctypes.POINTER(u64)], i32),
            "thr_peer_close": ([u64], i32),
            "thr_peer_free": ([u64], i32),
        }
        for name, (args, res) in sig.items():
            f = getattr(lib, name)
            f.argtypes, f.restype = args, res
        _lib = lib
    return _lib


def last_error() -> str:
    buf = ctypes.create_string_buffer(65536)
    library().thr_last_error(buf, len(buf))
    return buf.value.decode(errors="replace")


def check(status: int, what: str) -> None:
    if status:
        raise RunnerError(STAGES.get(status, "cuda"), f"{what}: {last_error()}")


def init(device: int = 0) -> None:
    """Make ``device`` current in this thread (every call: modules load into the current
    device's context, so a caller switching devices must not be left on the previous one)."""
    check(library().thr_init(device), f"thr_init({device})")


def device_info(device: int = 0) -> dict:
    init(device)
    sm, ma, mi = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    name = ctypes.create_string_buffer(256)
    check(library().thr_device_info(device, sm, ma, mi, name, 256), "thr_device_info")
    return {"sm_count": sm.value, "cc": (ma.value, mi.value), "name": name.value.decode()}


def _dims(v) -> ctypes.Array:
    v = list(v) + [1, 1, 1]
    return (ctypes.c_uint32 * 3)(*[int(x) for x in v[:3]])


OVERLAP_PREVIOUS = 1                                # THR_LAUNCH_OVERLAP_PREVIOUS
ENTRY = re.compile(r"^\s*\.(?:visible\s+)?\.entry\s+([A-Za-z_$][\w$]*)\s*\(", re.M)


@dataclass
class Function:
    module: "Module"
    name: str
    handle: int
    num_regs: int = 0
    max_threads: int = 0
    static_smem: int = 0
    local_bytes: int = 0

    def launch(self, grid, block, smem: int, ptrs: list[int], stream: int = 0, overlap: bool = False) -> None:
        """Launch on device pointers; ``overlap``: programmatic dependent launch (the kernel may
        begin during the stream's previous kernel -- only for kernels that wait for it before
        touching global data, ``LaunchPlan.pdl``)."""
        a = (ctypes.c_uint64 * max(1, len(ptrs)))(*[int(p) for p in ptrs])
        check(library().thr_launch_ex(self.handle, _dims(grid), _dims(block), int(smem), a, len(ptrs), int(stream),
                                      OVERLAP_PREVIOUS if overlap else 0),
              f"launch of {self.name}")


@dataclass
class Module:
    ptx: str
    handle: int
    log: str = ""
    sidecar: dict | None = None
    functions: dict = field(default_factory=dict)

    @property
    def entry_points(self) -> list[str]:
        return ENTRY.findall(self.ptx)

    def function(self, entry: str) -> Function:
        f = self.functions.get(entry)
        if f is None:
            h = ctypes.c_uint64()
            check(library().thr_get_function(self.handle, entry.encode(), ctypes.byref(h)), f"entry {entry}")
            r, t, s, lb = ctypes.c_int(), ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
            check(library().thr_function_attrs(h.value, r, t, s, lb), "thr_function_attrs")
            f = Function(self, entry, h.value, r.value, t.value, s.value, lb.value)
            self.functions[entry] = f
        return f

    def global_ptr(self, name: str) -> tuple[int, int]:
        p, n = ctypes.c_uint64(), ctypes.c_uint64()
        check(library().thr_module_global(self.handle, name.encode(), ctypes.byref(p), ctypes.byref(n)),
              f"module global {name}")
        return p.value, n.value

    def unload(self) -> None:
        if self.handle:
            library().thr_module_unload(self.handle)
            self.handle = 0


def load_module(ptx: str, device: int = 0) -> Module:
    init(device)
    h = ctypes.c_uint64()
    log = ctypes.create_string_buffer(16384)
    check(library().thr_module_load(ptx.encode(), ctypes.byref(h), log, len(log)), "PTX JIT")
    return Module(ptx, h.value, log.value.decode(errors="replace"), read_sidecar(ptx))


def compile_ptx(ptx: str, device: int = 0) -> dict:
    """POST /compile: assemble ``ptx``; never raises for a bad module."""
    try:
        mod = load_module(ptx, device)
    except RunnerError as e:
        return {"ok": False, "stage": e.stage, "stderr": e.message}
    regs = {}
    for entry in mod.entry_points:
        try:
            regs[entry] = mod.function(entry).num_regs
        except RunnerError as e:
            return {"ok": False, "stage": e.stage, "stderr": e.message}
    return {"ok": True, "entry_points": mod.entry_points, "registers": regs, "module": mod}


# ---- launch plans -----------------------------------------------------------

DTYPE_CODE = {"f16": 0, "bf16": 1, "f32": 2}


@dataclass
class LaunchPlan:
    grid: tuple
    block: tuple
    smem: int
    tuned: bool
    tmaps: list = field(default_factory=list)       # tensor-map specs the tuned launch reads
    tmap_ptrs: dict | None = None                   # {"global": name, "params": [...]}
    error_word: str | None = None                   # module global a kernel records wait time-outs in
    counters: list = field(default_factory=list)    # self-resetting arrival counters (module globals)
    pdl: bool = False                               # the tuned body waits (griddepcontrol.wait) before
                                                    # global accesses: launches may overlap the previous kernel
                                                    # (meta.json's too, unless the record says pdl_meta: false)
    align: dict = field(default_factory=dict)       # buffer -> the boundary, in bytes, that it has to start on


def plan_launch(module: Module, kmeta: dict, honour_meta: bool = False) -> LaunchPlan:
    """meta.json's geometry, or the tuned launch recorded in the PTX.  Tensor maps the IR itself
    declares (TmaDescriptor statements: the sidecar's ``ir_tmaps``) belong to every launch."""
    side = module.sidecar or {}
    ir_maps = list(side.get("ir_tmaps", []))
    counters = list(side.get("counters", []))
    if "grid" not in side or honour_meta:
        return LaunchPlan(tuple(kmeta["grid"]), tuple(kmeta["block"]), int(kmeta.get("smem_bytes", 0)), False,
                          ir_maps, None, side.get("error_word"), counters,
                          bool(side.get("pdl_meta", side.get("pdl", False))))
    return LaunchPlan(tuple(side["grid"]), tuple(side["block"]), int(side.get("smem_bytes", 0)), True,
                      list(side.get("tmaps", [])) + ir_maps, side.get("tmap_ptrs"), side.get("error_word"),
                      counters, bool(side.get("pdl", False)), dict(side.get("align", {})))


def encode_tensor_map(spec: dict, base: int) -> bytes:
    out = ctypes.create_string_buffer(128)
    dims = (ctypes.c_uint64 * 5)(*spec["dims"])
    strides = (ctypes.c_uint64 * 4)(*(spec.get("strides") or [0]))
    box = (ctypes.c_uint32 * 5)(*spec["box"])
    check(library().thr_tensor_map(out, DTYPE_CODE[spec["dtype"]], len(spec["dims"]), int(base), dims, strides,
                                   box, int(spec.get("swizzle", 0))), "tensor map")
    return out.raw


class TensorMaps:
    """The tensor maps of one tuned launch plan, for launches on device pointers: ``bind`` makes
    the module's tensor-map set for the given buffers current on a stream (encoding and uploading
    it, stream-ordered, when no set holds those buffers yet) and returns its index; ``launched``
    records that a launch reading the set was just issued on the stream, so that re-encoding the
    set later waits for it (thr_tmap_bind / thr_tmap_launched)."""

    def __init__(self, module: Module, plan: LaunchPlan, arg_order: list[str]):
        self.module, self.arg_order = module, list(arg_order)
        self.specs, self._names = _tmap_specs(plan, self.arg_order)
        self.n = len(plan.tmaps)
        sets = (module.sidecar or {}).get("tmap_sets")
        if sets is not None:                   # the ring the runner finds must be the one the kernel reads
            _, size = module.global_ptr(plan.tmaps[0]["global"])
            if size != sets * self.n * 128 or len({t["global"] for t in plan.tmaps}) != 1:
                raise RunnerError("lookup", f"tensor-map ring {plan.tmaps[0]['global']}: {size} bytes for "
                                            f"{sets} sets of {self.n} maps")
        self.table = plan.tmap_ptrs["global"].encode() if plan.tmap_ptrs else None
        self._args = (ctypes.c_uint64 * len(self.arg_order))()
        self._set = ctypes.c_int()

    def bind(self, ptrs: dict[str, int], stream: int = 0) -> int:
        for i, name in enumerate(self.arg_order):
            self._args[i] = ptrs[name]
        check(library().thr_tmap_bind(self.module.handle, self.specs, self.n, self.table, self._args,
                                      len(self.arg_order), int(stream), ctypes.byref(self._set)), "tensor maps")
        return self._set.value

    def launched(self, set_: int, stream: int = 0) -> None:
        check(library().thr_tmap_launched(self.module.handle, int(set_), int(stream)), "tensor maps")


class Launch:
    """One kernel's launches on device pointers.  What stays the same from call to call is a C record made
    once, so ``launch(ptrs, stream)`` packs the pointers and makes one C call (with its tensor maps'
    binding, when the plan has any).  ``plan``'s grid, block, shared memory and overlap are read again
    whenever they are replaced; a buffer that meta.json or the launch record wants aligned is refused when
    it is not."""

    def __init__(self, function: Function, plan: LaunchPlan, kmeta: dict, tmaps: TensorMaps | None):
        self.function, self.plan, self.order, self.tmaps = function, plan, tuple(kmeta["arg_order"]), tmaps
        n = len(self.order)
        self._get = operator.itemgetter(*self.order) if n > 1 else lambda ptrs: tuple(ptrs[x] for x in self.order)
        self._pack = struct.Struct(f"@{max(1, n)}Q").pack if n else lambda: bytes(8)
        align, own = {a["name"]: a.get("align", 0) for a in kmeta["args"]}, getattr(plan, "align", {})
        self._align = (ctypes.c_uint32 * max(1, n))(*[max(align.get(x, 0), own.get(x, 0)) for x in self.order])
        self._call = library().thr_launch_prepared
        self._geometry, self._descs = None, []

    def _prepare(self) -> None:
        plan, t = self.plan, self.tmaps
        d = ThrLaunchDesc(self.function.module.handle if t else 0, self.function.handle, _dims(plan.grid),
                          _dims(plan.block), int(plan.smem), OVERLAP_PREVIOUS if plan.pdl else 0, len(self.order))
        d.align = self._align
        if t is not None:
            d.tmaps, d.ntmaps, d.ptr_table = t.specs, t.n, t.table
        self._descs.append(d)                 # kept: a call in another thread may still be reading the last one
        self._at = ctypes.addressof(d)
        self._geometry = (plan.grid, plan.block, plan.smem, plan.pdl)

    def __call__(self, ptrs: dict[str, int], stream: int = 0) -> None:
        plan = self.plan
        if (plan.grid, plan.block, plan.smem, plan.pdl) != self._geometry:
            self._prepare()
        st = self._call(self._at, self._pack(*self._get(ptrs)), stream)
        if st:
            why = last_error()
            m = re.match(r"argument (\d+) at", why)
            if m:
                why = f"buffer {self.order[int(m[1])]!r}" + why[m.end() - 3:]
            raise RunnerError(STAGES.get(st, "cuda"), f"launch of {self.function.name}: {why}")


def read_error_word(module: Module, plan: LaunchPlan) -> int:
    """The kernel's error word (0: no bounded wait gave up and no guarded copy or MMA was skipped),
    or 0 if it has none."""
    if not plan.error_word:
        return 0
    dst, _ = module.global_ptr(plan.error_word)
    v = ctypes.c_uint32()
    check(library().thr_memcpy_dtoh(ctypes.byref(v), dst, 4), "error word")
    return v.value


def clear_error_word(module: Module, plan: LaunchPlan) -> None:
    """Zero the kernel's error word and the self-resetting arrival counters its family declares
    (``counters`` in the launch record).  A bounded wait that gave up can leave such a counter
    part-way through its count, and the next launch would then take the wrong K part of a tile
    as the last to arrive and add partials that were never written.  Call this after a launch
    whose error word was non-zero, before the module is launched again."""
    lib = library()
    names = ([plan.error_word] if plan.error_word else []) + list(plan.counters)
    for name in names:
        dst, size = module.global_ptr(name)
        zeros = ctypes.create_string_buffer(size)
        check(lib.thr_memcpy_htod(dst, zeros, size, 0), f"clear {name}")
    check(lib.thr_synchronize(), "clear error word")


def _tmap_specs(plan: LaunchPlan, arg_order: list[str]):
    specs = (ThrTmapSpec * max(1, len(plan.tmaps)))()
    names = []
    for i, t in enumerate(plan.tmaps):
        names.append(t["global"].encode())
        specs[i].global_ = names[-1]
        specs[i].arg = arg_order.index(t["param"])
        specs[i].dtype_code = DTYPE_CODE[t["dtype"]]
        specs[i].rank = len(t["dims"])
        specs[i].swizzle = int(t.get("swizzle", 0))
        for j, v in enumerate(t["dims"]):
            specs[i].dims[j] = v
        for j, v in enumerate(t.get("strides") or []):
            specs[i].strides[j] = v
        for j, v in enumerate(t["box"]):
            specs[i].box[j] = v
    return specs, names


def run(function: Function, plan: LaunchPlan, args: list[dict], warmup: int = 0, iters: int = 1,
        timeout_s: float = 20.0, stream: int = 0, arg_order: list[str] | None = None) -> dict:
    """POST /run on host buffers.  ``args``: dicts with ``array`` (numpy; outputs
    are written back into it), ``output`` (bool) and ``zero_each`` (bool), in
    the kernel's argument order (``arg_order`` names them; needed for tuned
    launches that read tensor maps)."""
    arr = (ThrArg * max(1, len(args)))()
    keep = []
    for i, a in enumerate(args):
        x = np.ascontiguousarray(a["array"])
        keep.append(x)
        arr[i].host = x.ctypes.data
        arr[i].nbytes = x.nbytes
        arr[i].kind = 1 if a.get("output") else 0
        arr[i].zero_each = 1 if a.get("zero_each") else 0
    med = ctypes.c_float()
    lib = library()
    if plan.tmaps:
        if arg_order is None:
            raise RunnerError("request", "a tuned launch with tensor maps needs the argument names")
        specs, _names = _tmap_specs(plan, arg_order)
        table = plan.tmap_ptrs["global"].encode() if plan.tmap_ptrs else None
        st = lib.thr_run_ex(function.module.handle, function.handle, _dims(plan.grid), _dims(plan.block),
                            int(plan.smem), arr, len(args), specs, len(plan.tmaps), table, int(warmup), int(iters),
                            float(timeout_s), ctypes.byref(med), int(stream))
    else:
        st = lib.thr_run(function.handle, _dims(plan.grid), _dims(plan.block), int(plan.smem), arr, len(args),
                         int(warmup), int(iters), float(timeout_s), ctypes.byref(med), int(stream))
    if st:
        return {"ok": False, "stage": STAGES.get(st, "cuda"), "stderr": last_error()}
    for a, x in zip(args, keep):
        if a.get("output") and x is not a["array"]:
            a["array"][...] = x
    err = read_error_word(function.module, plan)
    if err:
        return {"ok": False, "stage": "run", "stderr": f"kernel error word {err:#x} (a bounded wait gave up or a guarded copy was skipped)"}
    return {"ok": True, "median_us": float(med.value)}


class PreparedBatch:
    """Independent POST /run requests for thr_run_batch with their C descriptors built once, so a
    caller that repeats a batch (a serving loop, the e2e benchmark) pays no per-call Python setup.
    ``requests``: (function, plan, args, arg_order) tuples, ``args`` as for ``run``; pass pinned,
    C-contiguous host arrays for the copies to overlap and to be read and written in place (others
    are staged through private copies, refreshed on every run)."""

    def __init__(self, requests: list) -> None:
        self.n = len(requests)
        self.descs = (ThrRunDesc * max(1, self.n))()
        self._keep = []
        self._staged = []                       # (caller's array, private copy, is output)
        for r, (function, plan, args, arg_order) in enumerate(requests):
            arr = (ThrArg * max(1, len(args)))()
            for i, a in enumerate(args):
                x = np.ascontiguousarray(a["array"])
                if x is not a["array"]:
                    self._staged.append((a["array"], x, bool(a.get("output"))))
                self._keep.append(x)
                arr[i].host = x.ctypes.data
                arr[i].nbytes = x.nbytes
                arr[i].kind = 1 if a.get("output") else 0
                arr[i].zero_each = 1 if a.get("zero_each") else 0
            d = self.descs[r]
            d.module, d.function = function.module.handle, function.handle
            d.grid, d.block = _dims(plan.grid), _dims(plan.block)
            d.smem_bytes, d.nargs, d.args = int(plan.smem), len(args), arr
            if plan.tmaps:
                specs, names = _tmap_specs(plan, arg_order)
                table = plan.tmap_ptrs["global"].encode() if plan.tmap_ptrs else None
                d.tmaps, d.ntmaps, d.ptr_table = specs, len(plan.tmaps), table
                self._keep.append((specs, names, table))
            self._keep.append(arr)
        # one error-word read per module that has one
        seen, self._checks = set(), []
        for function, plan, _, _ in requests:
            if plan.error_word and function.module.handle not in seen:
                seen.add(function.module.handle)
                self._checks.append((function.module, plan))

    def run(self, timeout_s: float = 60.0) -> dict:
        for src, x, out in self._staged:
            if not out:
                x[...] = src
        st = library().thr_run_batch(self.descs, self.n, float(timeout_s))
        if st:
            return {"ok": False, "stage": STAGES.get(st, "cuda"), "stderr": last_error()}
        for src, x, out in self._staged:
            if out:
                src[...] = x
        for module, plan in self._checks:
            err = read_error_word(module, plan)
            if err:
                return {"ok": False, "stage": "run", "stderr": f"kernel error word {err:#x} (a bounded wait gave up or a guarded copy was skipped)"}
        return {"ok": True}


def run_batch(requests: list, timeout_s: float = 60.0) -> dict:
    """Several independent POST /run requests with their copies and launches overlapped
    (thr_run_batch), prepared and run once; see ``PreparedBatch``."""
    return PreparedBatch(requests).run(timeout_s)


def release() -> None:
    if _lib is not None:
        _lib.thr_release_buffers()
