"""ctypes binding of include/polar_hip.h (the device library's C ABI).

Every function of the header is bound with its exact signature; a non-zero
status raises ``PolarHipError`` carrying ``polar_hip_last_error()``.  The
``Device`` class is a thin convenience over the raw calls for tests and the
benchmark: it moves numpy arrays in and out of pool memory and enqueues the
builtin-operation kernels.  There is no fallback path: a missing library or a
missing GPU raises.
"""
import ctypes as C
import os

import numpy as np

from . import LIB_DEVICE


class PolarHipError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(f"polar_hip status {status}: {message}")
        self.status = status


class DeviceInfo(C.Structure):
    _fields_ = [
        ("name", C.c_char * 256),
        ("arch", C.c_char * 64),
        ("ordinal", C.c_int),
        ("compute_units", C.c_int),
        ("clock_khz", C.c_int),
        ("memory_clock_khz", C.c_int),
        ("memory_bus_bits", C.c_int),
        ("lds_bytes_per_block", C.c_int),
        ("l2_bytes", C.c_int),
        ("pci_bus_id", C.c_int),
        ("hbm_bytes", C.c_uint64),
    ]


class PoolStats(C.Structure):
    _fields_ = [
        ("bytes_in_use", C.c_uint64),
        ("bytes_cached", C.c_uint64),
        ("device_allocs", C.c_uint64),
        ("pool_hits", C.c_uint64),
    ]


class AdamWTensor(C.Structure):
    _fields_ = [
        ("param", C.c_void_p),
        ("grad", C.c_void_p),
        ("m", C.c_void_p),
        ("v", C.c_void_p),
        ("master", C.c_void_p),
        ("m_scale", C.c_void_p),
        ("v_scale", C.c_void_p),
        ("count", C.c_uint64),
        ("first", C.c_uint64),
        ("weight_decay", C.c_double),
    ]


class AdamWConfig(C.Structure):
    _fields_ = [
        ("param_type", C.c_int),
        ("grad_type", C.c_int),
        ("state_bits", C.c_int),
        ("seed", C.c_uint32),
        ("step", C.c_int64),
        ("lr", C.c_double),
        ("beta1", C.c_double),
        ("beta2", C.c_double),
        ("eps", C.c_double),
        ("grad_scale", C.c_double),
    ]


TYPES = {"f32": 0, "f16": 1, "bf16": 2}         # polar_hip_type
INDEX_TYPES = {"i32": 0, "i64": 1, "f32": 2}    # polar_hip_index_type
STATE_BITS = {"f32": 32, "8bit": 8}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}         # bytes of an element
INDEX_SIZES = {"i32": 4, "i64": 8, "f32": 4}
LOGPROB_MAX_TOP = 32
ADAMW_BLOCK = 256

_vp = C.c_void_p
_u64 = C.c_uint64
_u32 = C.c_uint32
_f = C.c_float
_i = C.c_int

# name -> (restype, argtypes); one entry per declaration in include/polar_hip.h
SIGNATURES = {
    "polar_hip_last_error": (C.c_char_p, []),
    "polar_hip_version": (C.c_char_p, []),
    "polar_hip_device_count": (_i, [C.POINTER(_i)]),
    "polar_hip_device_open": (_i, [_i, C.POINTER(_vp)]),
    "polar_hip_device_close": (_i, [_vp]),
    "polar_hip_device_get_info": (_i, [_vp, C.POINTER(DeviceInfo)]),
    "polar_hip_device_synchronize": (_i, [_vp]),
    "polar_hip_alloc": (_i, [_vp, _u64, C.POINTER(_vp)]),
    "polar_hip_free": (_i, [_vp, _vp]),
    "polar_hip_pool_trim": (_i, [_vp]),
    "polar_hip_pool_get_stats": (_i, [_vp, C.POINTER(PoolStats)]),
    "polar_hip_copy_to_device": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_copy_to_host": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_host_alloc": (_i, [_vp, _u64, C.POINTER(_vp)]),
    "polar_hip_host_free": (_i, [_vp]),
    "polar_hip_host_quiesce": (_i, [_vp]),
    "polar_hip_event_record": (_i, [_vp, C.POINTER(_vp)]),
    "polar_hip_event_synchronize": (_i, [_vp]),
    "polar_hip_event_query": (_i, [_vp, C.POINTER(_i)]),
    "polar_hip_stream_wait_event": (_i, [_vp, _vp]),
    "polar_hip_event_elapsed_ms": (_i, [_vp, _vp, C.POINTER(_f)]),
    "polar_hip_time_next_kernel": (_i, [_vp, C.POINTER(_vp), C.POINTER(_vp)]),
    "polar_hip_event_release": (_i, [_vp]),
    "polar_hip_fadd": (_i, [_vp, _vp, _f, _vp, _f, _vp, _u64]),
    "polar_hip_fmul": (_i, [_vp, _vp, _vp, _vp, _u64]),
    "polar_hip_fdivide": (_i, [_vp, _vp, _vp, _vp, _u64]),
    "polar_hip_fsigmoid": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_flogloss": (_i, [_vp, _vp, _vp, _vp, _u64]),
    "polar_hip_fmulconcat": (_i, [_vp, _vp, _vp, _vp, _u64]),
    "polar_hip_fcopy": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_ffill": (_i, [_vp, _f, _vp, _u64]),
    "polar_hip_ftranspose": (_i, [_vp, _vp, _vp, _u64, _u64]),
    "polar_hip_fmatmul": (_i, [_vp, _i, _i, _vp, _vp, _vp, _u64, _u64, _u64]),
    "polar_hip_fmatmul_plan": (_i, [_vp, _u64, _u64, _u64, C.POINTER(_i), C.POINTER(C.c_uint32),
                                    C.POINTER(C.c_uint32)]),
    "polar_hip_fmatmul_with_plan": (_i, [_vp, _i, _i, _vp, _vp, _vp, _u64, _u64, _u64, _i, C.c_uint32]),
    "polar_hip_module_load": (_i, [_vp, _vp, _u64, C.POINTER(_vp)]),
    "polar_hip_module_unload": (_i, [_vp, _vp]),
    "polar_hip_module_has_kernel": (_i, [_vp, C.c_char_p, C.POINTER(_i)]),
    "polar_hip_module_launch": (_i, [_vp, _vp, C.c_char_p, C.POINTER(C.c_uint32), C.POINTER(C.c_uint32),
                                     C.POINTER(_vp)]),
    "polar_hip_frelu": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_fsoftmax": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_fsoftmax_static": (_i, [_vp, _vp, _vp, _u64]),
    "polar_hip_fconv2d": (_i, [_vp, _vp, _vp, _vp, _u64, _u64, _u64, _u64]),
    "polar_hip_fpool": (_i, [_vp, _vp, _vp, _u64, _u64, _u64, _u64, _u64, _u64]),
    "polar_hip_fpool_plan": (_i, [_u64, _u64, _u64, _u64, _u64, _u64, _i, C.POINTER(C.c_int), C.POINTER(C.c_uint32),
                                  C.POINTER(C.c_uint32)]),
    "polar_hip_fmatmul_fsigmoid": (_i, [_vp, _i, _i, _vp, _vp, _vp, _u64, _u64, _u64]),
    "polar_hip_fmatmul_fadd_fsigmoid": (_i, [_vp, _i, _i, _vp, _vp, _f, _vp, _f, _vp, _u64, _u64, _u64]),
    "polar_hip_fsigmoid_flogloss": (_i, [_vp, _vp, _vp, _vp, _u64]),
    "polar_hip_flayernorm": (_i, [_vp, _i, _vp, _u64, _i, _vp, _vp, _f, _vp, _u64, _vp, _vp, _u64, _u64]),
    "polar_hip_flayernorm_grad": (_i, [_vp, _i, _vp, _u64, _vp, _u64, _i, _vp, _vp, _vp, _f, _vp, _u64, _vp, _vp,
                                       _u64, _u64]),
    "polar_hip_flogprob": (_i, [_vp, _i, _vp, _u64, _i, _vp, _f, _vp, _vp, _vp, _u32, _vp, _vp, _u64, _u64]),
    "polar_hip_flogprob_grad": (_i, [_vp, _i, _vp, _u64, _i, _vp, _f, _vp, _vp, _vp, _vp, _vp, _u64, _u64, _u64]),
    "polar_hip_fadamw": (_i, [_vp, C.POINTER(AdamWConfig), C.POINTER(AdamWTensor), _u64]),
}

_lib = None


def load_library(path=LIB_DEVICE):
    """Load libpolar_hip.so and bind every declared symbol.  Raises if the
    library or any symbol is missing."""
    global _lib
    if _lib is not None and path == LIB_DEVICE:
        return _lib
    if not os.path.exists(path):
        raise FileNotFoundError(
            f"{path} is not built; run __graft_entry__.build() (hipcc, gfx950)")
    lib = C.CDLL(path, mode=C.RTLD_GLOBAL)
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(lib, name)  # AttributeError if the symbol is absent
        fn.restype = res
        fn.argtypes = args
    if path == LIB_DEVICE:
        _lib = lib
    return lib


def _check(lib, status):
    if status != 0:
        raise PolarHipError(status, lib.polar_hip_last_error().decode())


def _ptr(x, name, nbytes, ordinal):
    """Device address of a Buffer, of a tensor of another library on the same GPU (anything with data_ptr()), or of
    a plain address; None stays None.  The device's stream is its own: work of another library on such a tensor is
    waited for before the call, and the call before that library uses the tensor again.  A tensor that says where it
    lies (get_device()) and what it holds (nbytes) is refused on another device, or with less than `nbytes` bytes: a
    kernel would access memory that is not its own."""
    if x is None:
        return None
    kind = x.__class__
    if kind is int:
        return x
    if kind is Buffer:
        return x.ptr
    try:
        if x.get_device() == ordinal and x.nbytes >= nbytes:
            return x.data_ptr()
    except AttributeError:
        if isinstance(x, int):
            return x
        at = getattr(x, "ptr", None)
        return x.data_ptr() if at is None else at
    _check_place(x, name, x.get_device(), ordinal)
    if x.nbytes < nbytes:
        raise ValueError(f"{name} holds {x.nbytes} bytes, {nbytes} are needed (its dtype, rows or columns?)")
    return x.data_ptr()


def _check_place(x, name, where, ordinal):
    """Refuses a tensor that does not lie on device `ordinal`; pinned host memory is accessible from all of them."""
    if where < 0:
        pinned = getattr(x, "is_pinned", None)
        if pinned is None or not pinned():
            raise TypeError(f"{name} is not in device memory")
    elif where != ordinal:
        raise TypeError(f"{name} lies on device {where}, the call is made on device {ordinal}")


def adamw_tensors(tensors):
    """The list of tensors that Device.fadamw takes, from dicts with the fields of polar_hip_adamw_tensor (those left
    out or None are null; weight_decay is 0).  A training program makes it once; it keeps what it was given alive.
    Where a gradient moves from step to step, its address is put into the list: plan[i].grad = gradient.data_ptr()."""
    table = (AdamWTensor * len(tensors))()
    # for fadamw, which knows device and types: a field for each device that a tensor lies on, and for each field the
    # fewest bytes that one of its tensors holds per element (of the scales, per block)
    table.kept, table.places, table.room = [], {}, {}
    for entry, t in zip(table, tensors):
        count = int(t.get("count", 0))
        for name, value in t.items():
            if name in ("count", "first"):
                setattr(entry, name, int(value))
            elif name == "weight_decay":
                entry.weight_decay = value
            elif name in ("param", "grad", "m", "v", "master", "m_scale", "v_scale"):
                where = value.get_device() if hasattr(value, "get_device") and hasattr(value, "nbytes") else None
                setattr(entry, name, _ptr(value, name, 0, where))
                if value is None or isinstance(value, int):
                    continue
                table.kept.append(value)
                if where is None:
                    continue
                if where < 0:
                    _check_place(value, name, where, where)
                else:
                    table.places[where] = name
                units = -(-count // ADAMW_BLOCK) if name.endswith("scale") else count
                if units:
                    table.room[name] = min(table.room.get(name, 1 << 62), value.nbytes // units)
            else:
                raise KeyError(f"no field {name} in a tensor of fadamw")
    return table


def fpool_plan(height, width, window, stride, input_aligned=True):
    """(kernel, band rows, LDS bytes) polar_hip_fpool would use: kernel 0 = taps
    from memory, 1 = non-overlapping square windows, 2 = window staged in LDS,
    3 = waves marching down strips (square windows of 4 and 5).  Needs no GPU."""
    lib = load_library()
    kernel, band, lds = _i(0), C.c_uint32(0), C.c_uint32(0)
    _check(lib, lib.polar_hip_fpool_plan(height, width, window[0], window[1], stride[0], stride[1],
                                         int(bool(input_aligned)), C.byref(kernel), C.byref(band), C.byref(lds)))
    return kernel.value, band.value, lds.value


def device_count():
    lib = load_library()
    n = _i(0)
    _check(lib, lib.polar_hip_device_count(C.byref(n)))
    return n.value


class Buffer:
    """A block of pool memory on one device holding `count` fp32 elements."""

    def __init__(self, dev, count, ptr, offset_bytes=0):
        self.dev = dev
        self.count = int(count)
        self._base = ptr
        self.ptr = ptr + offset_bytes
        self.nbytes = self.count * 4

    def free(self):
        if self._base is not None:
            self.dev._free(self._base)
            self._base = None

    def upload(self, arr):
        arr = np.ascontiguousarray(arr, dtype=np.float32)
        assert arr.size == self.count, (arr.size, self.count)
        self.dev.copy_to_device(self.ptr, arr.ctypes.data, self.nbytes)
        return self

    def download(self, shape=None):
        out = np.empty(self.count, dtype=np.float32)
        self.dev.copy_to_host(out.ctypes.data, self.ptr, self.nbytes)
        return out if shape is None else out.reshape(shape)


class Event:
    def __init__(self, dev, handle):
        self.dev = dev
        self.handle = handle

    def synchronize(self):
        _check(self.dev.lib, self.dev.lib.polar_hip_event_synchronize(self.handle))

    def done(self):
        d = _i(0)
        _check(self.dev.lib, self.dev.lib.polar_hip_event_query(self.handle, C.byref(d)))
        return bool(d.value)

    def elapsed_ms(self, later):
        ms = _f(0)
        _check(self.dev.lib, self.dev.lib.polar_hip_event_elapsed_ms(
            self.handle, later.handle, C.byref(ms)))
        return ms.value

    def release(self):
        _check(self.dev.lib, self.dev.lib.polar_hip_event_release(self.handle))
        self.handle = None


class Device:
    """One opened GPU (stream + memory pool)."""

    def __init__(self, ordinal=0):
        self.lib = load_library()
        h = _vp()
        _check(self.lib, self.lib.polar_hip_device_open(ordinal, C.byref(h)))
        self.handle = h
        self.ordinal = ordinal

    # -- lifetime -----------------------------------------------------------
    def close(self):
        if self.handle is not None:
            _check(self.lib, self.lib.polar_hip_device_close(self.handle))
            self.handle = None

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def info(self):
        inf = DeviceInfo()
        _check(self.lib, self.lib.polar_hip_device_get_info(self.handle, C.byref(inf)))
        return inf

    def synchronize(self):
        _check(self.lib, self.lib.polar_hip_device_synchronize(self.handle))

    # -- memory -------------------------------------------------------------
    def alloc_bytes(self, nbytes):
        p = _vp()
        _check(self.lib, self.lib.polar_hip_alloc(self.handle, nbytes, C.byref(p)))
        return p.value

    def _free(self, ptr):
        _check(self.lib, self.lib.polar_hip_free(self.handle, ptr))

    def empty(self, count, misalign_floats=0):
        """fp32 buffer of `count` elements; `misalign_floats` shifts the
        start by that many elements past the 256-byte aligned block."""
        ptr = self.alloc_bytes((int(count) + misalign_floats) * 4)
        return Buffer(self, count, ptr, misalign_floats * 4)

    def array(self, arr, misalign_floats=0):
        arr = np.ascontiguousarray(arr, dtype=np.float32)
        return self.empty(arr.size, misalign_floats).upload(arr)

    def copy_to_device(self, dst, src_host, nbytes):
        _check(self.lib, self.lib.polar_hip_copy_to_device(self.handle, dst, src_host, nbytes))

    def copy_to_host(self, dst_host, src, nbytes):
        _check(self.lib, self.lib.polar_hip_copy_to_host(self.handle, dst_host, src, nbytes))

    def host_alloc(self, nbytes):
        """Pinned host memory that the copy calls move to and from directly."""
        p = _vp()
        _check(self.lib, self.lib.polar_hip_host_alloc(self.handle, nbytes, C.byref(p)))
        return p.value

    def host_free(self, ptr):
        _check(self.lib, self.lib.polar_hip_host_free(ptr))

    def host_quiesce(self, ptr):
        _check(self.lib, self.lib.polar_hip_host_quiesce(ptr))

    def pool_stats(self):
        st = PoolStats()
        _check(self.lib, self.lib.polar_hip_pool_get_stats(self.handle, C.byref(st)))
        return st

    def pool_trim(self):
        _check(self.lib, self.lib.polar_hip_pool_trim(self.handle))

    # -- events -------------------------------------------------------------
    def record(self):
        h = _vp()
        _check(self.lib, self.lib.polar_hip_event_record(self.handle, C.byref(h)))
        return Event(self, h)

    def time_next_kernel(self):
        """(start, stop) events that take the next kernel's own begin and end."""
        s, e = _vp(), _vp()
        _check(self.lib, self.lib.polar_hip_time_next_kernel(self.handle, C.byref(s), C.byref(e)))
        return Event(self, s), Event(self, e)

    def wait_event(self, evt):
        _check(self.lib, self.lib.polar_hip_stream_wait_event(self.handle, evt.handle))

    # -- builtin operations (asynchronous) ------------------------------------
    def fadd(self, a, scale_a, b, scale_b, c, n=None):
        n = c.count if n is None else n
        _check(self.lib, self.lib.polar_hip_fadd(self.handle, a.ptr, scale_a, b.ptr, scale_b, c.ptr, n))

    def fmul(self, a, b, c, n=None):
        n = c.count if n is None else n
        _check(self.lib, self.lib.polar_hip_fmul(self.handle, a.ptr, b.ptr, c.ptr, n))

    def fdivide(self, num, den, out, n=None):
        n = out.count if n is None else n
        _check(self.lib, self.lib.polar_hip_fdivide(self.handle, num.ptr, den.ptr, out.ptr, n))

    def fsigmoid(self, x, out, n=None):
        n = out.count if n is None else n
        _check(self.lib, self.lib.polar_hip_fsigmoid(self.handle, x.ptr, out.ptr, n))

    def flogloss(self, pred, truth, out, n=None):
        n = out.count if n is None else n
        _check(self.lib, self.lib.polar_hip_flogloss(self.handle, pred.ptr, truth.ptr, out.ptr, n))

    def fmulconcat(self, grad, local, out, n=None):
        n = out.count if n is None else n
        _check(self.lib, self.lib.polar_hip_fmulconcat(self.handle, grad.ptr, local.ptr, out.ptr, n))

    def fcopy(self, src, dst, n=None):
        n = dst.count if n is None else n
        _check(self.lib, self.lib.polar_hip_fcopy(self.handle, src.ptr, dst.ptr, n))

    def ffill(self, pattern, out, n=None):
        n = out.count if n is None else n
        _check(self.lib, self.lib.polar_hip_ffill(self.handle, pattern, out.ptr, n))

    def ftranspose(self, src, dst, rows, cols):
        _check(self.lib, self.lib.polar_hip_ftranspose(self.handle, src.ptr, dst.ptr, rows, cols))

    def frelu(self, x, out, n=None):
        _check(self.lib, self.lib.polar_hip_frelu(self.handle, x.ptr, out.ptr, out.count if n is None else n))

    def fsoftmax(self, x, out, n=None):
        _check(self.lib, self.lib.polar_hip_fsoftmax(self.handle, x.ptr, out.ptr, out.count if n is None else n))

    def fsoftmax_static(self, x, out, n=None):
        _check(self.lib, self.lib.polar_hip_fsoftmax_static(self.handle, x.ptr, out.ptr, out.count if n is None else n))

    def fconv2d(self, x, kernel, out, height, width, kernel_height, kernel_width):
        _check(self.lib, self.lib.polar_hip_fconv2d(self.handle, x.ptr, kernel.ptr, out.ptr, height, width,
                                                    kernel_height, kernel_width))

    def fpool(self, x, out, height, width, window, stride):
        _check(self.lib, self.lib.polar_hip_fpool(self.handle, x.ptr, out.ptr, height, width,
                                                  window[0], window[1], stride[0], stride[1]))

    def fmatmul_fsigmoid(self, trans_a, trans_b, a, b, out, m, n, k):
        _check(self.lib, self.lib.polar_hip_fmatmul_fsigmoid(self.handle, int(trans_a), int(trans_b), a.ptr, b.ptr,
                                                             out.ptr, m, n, k))

    def fmatmul_fadd_fsigmoid(self, trans_a, trans_b, a, b, scale_product, bias, scale_bias, out, m, n, k):
        _check(self.lib, self.lib.polar_hip_fmatmul_fadd_fsigmoid(self.handle, int(trans_a), int(trans_b), a.ptr,
                                                                  b.ptr, scale_product, bias.ptr, scale_bias,
                                                                  out.ptr, m, n, k))

    def fsigmoid_flogloss(self, x, truth, out, n=None):
        _check(self.lib, self.lib.polar_hip_fsigmoid_flogloss(self.handle, x.ptr, truth.ptr, out.ptr,
                                                              out.count if n is None else n))

    def fmatmul_plan(self, m, n, k):
        """(tile configuration or -1, splits, (tile M, tile N, tile K)) the planner picks."""
        cfg, splits, tile = _i(0), C.c_uint32(0), (C.c_uint32 * 3)()
        _check(self.lib, self.lib.polar_hip_fmatmul_plan(self.handle, m, n, k, C.byref(cfg), C.byref(splits), tile))
        return cfg.value, splits.value, tuple(tile)

    def fmatmul_with_plan(self, trans_a, trans_b, a, b, c, m, n, k, tile_config, splits):
        _check(self.lib, self.lib.polar_hip_fmatmul_with_plan(
            self.handle, int(bool(trans_a)), int(bool(trans_b)), a.ptr, b.ptr, c.ptr, m, n, k, tile_config, splits))

    def fmatmul(self, trans_a, trans_b, a, b, c, m, n, k):
        _check(self.lib, self.lib.polar_hip_fmatmul(
            self.handle, int(bool(trans_a)), int(bool(trans_b)), a.ptr, b.ptr, c.ptr, m, n, k))

    # -- operators of a language model's training step and sampling loop (asynchronous) --
    # tensors are Buffers, tensors of another library, or device addresses (_ptr)
    def flayernorm(self, x, weight, bias, out, rows, cols, eps=1e-5, mean=None, rstd=None, dtype="f32",
                   param_dtype="f32", x_stride=None, out_stride=None):
        at, whole, params, stats = self.ordinal, rows * cols * SIZES[dtype], cols * SIZES[param_dtype], rows * 4
        _check(self.lib, self.lib.polar_hip_flayernorm(
            self.handle, TYPES[dtype], _ptr(x, "x", whole, at), cols if x_stride is None else x_stride,
            TYPES[param_dtype], _ptr(weight, "weight", params, at), _ptr(bias, "bias", params, at), eps,
            _ptr(out, "out", whole, at), cols if out_stride is None else out_stride, _ptr(mean, "mean", stats, at),
            _ptr(rstd, "rstd", stats, at), rows, cols))

    def flayernorm_grad(self, grad, x, weight, dx, dweight, dbias, rows, cols, eps=1e-5, mean=None, rstd=None,
                        dtype="f32", param_dtype="f32", grad_stride=None, x_stride=None, dx_stride=None):
        at, whole, params, stats = self.ordinal, rows * cols * SIZES[dtype], cols * SIZES[param_dtype], rows * 4
        _check(self.lib, self.lib.polar_hip_flayernorm_grad(
            self.handle, TYPES[dtype], _ptr(grad, "grad", whole, at), cols if grad_stride is None else grad_stride,
            _ptr(x, "x", whole, at), cols if x_stride is None else x_stride, TYPES[param_dtype],
            _ptr(weight, "weight", params, at), _ptr(mean, "mean", stats, at), _ptr(rstd, "rstd", stats, at), eps,
            _ptr(dx, "dx", whole, at), cols if dx_stride is None else dx_stride, _ptr(dweight, "dweight", params, at),
            _ptr(dbias, "dbias", params, at), rows, cols))

    def flogprob(self, logits, tokens, logprob, rows, cols, scale=1.0, stats=None, entropy=None, top=0, top_index=None,
                 top_logprob=None, dtype="f32", token_dtype="i64", stride=None):
        at, each, best = self.ordinal, rows * 4, rows * top * 4
        _check(self.lib, self.lib.polar_hip_flogprob(
            self.handle, TYPES[dtype], _ptr(logits, "logits", rows * cols * SIZES[dtype], at),
            cols if stride is None else stride, INDEX_TYPES[token_dtype],
            _ptr(tokens, "tokens", rows * INDEX_SIZES[token_dtype], at), scale, _ptr(logprob, "logprob", each, at),
            _ptr(stats, "stats", 2 * each, at), _ptr(entropy, "entropy", each, at), top,
            _ptr(top_index, "top_index", best, at), _ptr(top_logprob, "top_logprob", best, at), rows, cols))

    def flogprob_grad(self, logits, tokens, stats, dlogprob, dlogits, rows, cols, scale=1.0, entropy=None,
                      dentropy=None, dtype="f32", token_dtype="i64", stride=None, dlogits_stride=None):
        at, each, whole = self.ordinal, rows * 4, rows * cols * SIZES[dtype]
        _check(self.lib, self.lib.polar_hip_flogprob_grad(
            self.handle, TYPES[dtype], _ptr(logits, "logits", whole, at), cols if stride is None else stride,
            INDEX_TYPES[token_dtype], _ptr(tokens, "tokens", rows * INDEX_SIZES[token_dtype], at), scale,
            _ptr(stats, "stats", 2 * each, at), _ptr(dlogprob, "dlogprob", each, at),
            _ptr(entropy, "entropy", each, at), _ptr(dentropy, "dentropy", each, at),
            _ptr(dlogits, "dlogits", whole, at), cols if dlogits_stride is None else dlogits_stride, rows, cols))

    def fadamw(self, tensors, step, lr, beta1=0.9, beta2=0.999, eps=1e-8, grad_scale=1.0, seed=0, dtype="f32",
               grad_dtype="f32", state_dtype="f32"):
        """`tensors`: what adamw_tensors() made."""
        for where, name in getattr(tensors, "places", {}).items():
            _check_place(None, name, where, self.ordinal)
        state, scale = (1, 4) if state_dtype == "8bit" else (4, 0)
        need = dict(param=SIZES[dtype], grad=SIZES[grad_dtype], m=state, v=state, master=0 if dtype == "f32" else 4,
                    m_scale=scale, v_scale=scale)
        for name, room in getattr(tensors, "room", {}).items():
            if room < need[name]:
                raise ValueError(f"a tensor's {name} is too short: {room} bytes for each of its elements or blocks, "
                                 f"{need[name]} are needed")
        config = AdamWConfig(TYPES[dtype], TYPES[grad_dtype], STATE_BITS[state_dtype], seed, step, lr, beta1, beta2, eps,
                             grad_scale)
        _check(self.lib, self.lib.polar_hip_fadamw(self.handle, C.byref(config), tensors, len(tensors)))
