"""Python binding of the B200 tt-foil C-ABI (include/foil_c.h, lib/libfoil.so).

Two layers, matching the C header:

* ``Device`` / ``Kernel`` / ``Buffer`` mirror tt-foil's host API
  (open_device, allocate_buffer, write/read_buffer, load_kernel,
  set_runtime_args, register_cbs, execute, make_noc_*_addr); every failure
  raises :class:`FoilError` with the library's message, as the reference
  raises std::runtime_error.
* ``tilize`` / ``untilize`` / ``tile_copy`` / ``add_tiles`` / ``relu_tiles`` /
  ``bias_add_tiles`` / ``matmul_tiles`` run the CUDA kernels on tensors that
  already live on the GPU (torch CUDA tensors or raw device pointers), on the
  current torch stream.  ``w4_*`` (products of a few rows with 4-bit weights),
  ``block_norm`` (the norms around a residual block) and ``embed_rows``, with
  their gradients, do the same for row-major tensors.

There is no fallback: if lib/libfoil.so is missing or was built for another
GPU, importing or calling this module raises.
"""
import ctypes
import os

_HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(_HERE)
LIB_DIR = os.path.join(ROOT, "lib")
PROGRAMS_DIR = os.path.join(ROOT, "programs")
LIB_PATH = os.path.join(LIB_DIR, "libfoil.so")

FOIL_OK = 0
STATUS_NAMES = {1: "INVALID", 2: "OOM", 3: "NOT_FOUND", 4: "CUDA", 5: "TIMEOUT",
                6: "UNSUPPORTED", 7: "DEVICE"}
LOC_L1, LOC_DRAM = 0, 1
BRISC, NCRISC, TRISC0, TRISC1, TRISC2 = range(5)


class FoilError(RuntimeError):
    def __init__(self, status, message):
        super().__init__(message)
        self.status = status


class foil_core(ctypes.Structure):
    _fields_ = [("x", ctypes.c_uint32), ("y", ctypes.c_uint32)]


class foil_buffer(ctypes.Structure):
    _fields_ = [("location", ctypes.c_int32), ("reserved", ctypes.c_uint32),
                ("device_addr", ctypes.c_uint64), ("size_bytes", ctypes.c_uint64),
                ("core", foil_core)]


class foil_risc_binary(ctypes.Structure):
    _fields_ = [("risc", ctypes.c_int32), ("elf_path", ctypes.c_char_p)]


class foil_cb_config(ctypes.Structure):
    _fields_ = [("cb_index", ctypes.c_uint8), ("fifo_addr", ctypes.c_uint64),
                ("fifo_size", ctypes.c_uint32), ("num_pages", ctypes.c_uint32),
                ("page_size", ctypes.c_uint32)]


# Exported C-ABI symbols with their signatures (restype, argtypes).
_P = ctypes.c_void_p
_U16P = ctypes.c_void_p
_U32, _I32, _U64, _F32 = ctypes.c_uint32, ctypes.c_int32, ctypes.c_uint64, ctypes.c_float
SIGNATURES = {
    "foil_last_error": (ctypes.c_char_p, []),
    "foil_version": (ctypes.c_char_p, []),
    "foil_open_device": (ctypes.c_int, [ctypes.c_int, ctypes.c_char_p, ctypes.POINTER(foil_core),
                                        ctypes.c_size_t, ctypes.POINTER(_P)]),
    "foil_close_device": (ctypes.c_int, [_P]),
    "foil_allocate_buffer": (ctypes.c_int, [_P, ctypes.c_int32, ctypes.c_uint64, foil_core,
                                            ctypes.POINTER(foil_buffer)]),
    "foil_free_buffer": (ctypes.c_int, [_P, ctypes.POINTER(foil_buffer)]),
    "foil_write_buffer": (ctypes.c_int, [_P, ctypes.POINTER(foil_buffer), _P, ctypes.c_uint64]),
    "foil_read_buffer": (ctypes.c_int, [_P, ctypes.POINTER(foil_buffer), _P, ctypes.c_uint64]),
    "foil_load_kernel": (ctypes.c_int, [_P, ctypes.POINTER(foil_risc_binary), ctypes.c_size_t,
                                        foil_core, ctypes.POINTER(_P)]),
    "foil_release_kernel": (ctypes.c_int, [_P]),
    "foil_set_runtime_args": (ctypes.c_int, [_P, _P, ctypes.c_int32,
                                             ctypes.POINTER(ctypes.c_uint32), ctypes.c_size_t]),
    "foil_register_cbs": (ctypes.c_int, [_P, _P, ctypes.POINTER(foil_cb_config), ctypes.c_size_t]),
    "foil_execute": (ctypes.c_int, [_P, ctypes.POINTER(_P), ctypes.c_size_t, ctypes.c_int32]),
    "foil_make_noc_unicast_addr": (ctypes.c_int, [_P, foil_core, ctypes.c_uint64,
                                                  ctypes.POINTER(ctypes.c_uint64)]),
    "foil_make_noc_dram_addr": (ctypes.c_int, [_P, ctypes.c_uint64, ctypes.POINTER(ctypes.c_uint64)]),
    "foil_buffer_device_ptr": (ctypes.c_int, [_P, ctypes.POINTER(foil_buffer), ctypes.POINTER(_P)]),
    "foil_launch_count": (ctypes.c_uint64, []),
    "foil_tilize_dev": (ctypes.c_int, [_U16P, _U16P, ctypes.c_uint32, ctypes.c_uint32, _P]),
    "foil_untilize_dev": (ctypes.c_int, [_U16P, _U16P, ctypes.c_uint32, ctypes.c_uint32, _P]),
    "foil_tile_copy_dev": (ctypes.c_int, [_P, _P, ctypes.c_uint64, _P]),
    "foil_add_tiles_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, ctypes.c_uint64, _P]),
    "foil_relu_tiles_dev": (ctypes.c_int, [_U16P, _U16P, ctypes.c_uint64, _P]),
    "foil_bias_add_tiles_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, ctypes.c_uint32,
                                               ctypes.c_uint32, _P]),
    "foil_matmul_tiles_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, ctypes.c_uint32, ctypes.c_uint32,
                                             ctypes.c_uint32, _U16P, ctypes.c_int32, _P]),
    "foil_device_error_dev": (ctypes.c_int, [_P, ctypes.POINTER(ctypes.c_uint32)]),
    "foil_conv2d_nhwc_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, _U16P] + [ctypes.c_uint32] * 9 +
                             [ctypes.c_int32, _P]),
    "foil_matmul_tiles_noalloc_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, ctypes.c_uint32,
                                                     ctypes.c_uint32, ctypes.c_uint32, _U16P,
                                                     ctypes.c_int32, _P,
                                                     ctypes.POINTER(ctypes.c_uint32)]),
    "foil_matmul_tiles_host": (ctypes.c_int, [ctypes.c_int32, _U16P, _U16P, _U16P, ctypes.c_uint32,
                                              ctypes.c_uint32, ctypes.c_uint32, _U16P, ctypes.c_int32,
                                              ctypes.c_uint32]),
    "foil_conv2d_nhwc_host": (ctypes.c_int, [ctypes.c_int32, _U16P, _U16P, _U16P, _U16P] +
                              [ctypes.c_uint32] * 9 + [ctypes.c_int32, ctypes.c_uint32]),
    "foil_host_pipeline_release": (ctypes.c_int, [ctypes.c_int32]),
    "foil_matmul_tiles_gather_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, ctypes.POINTER(_P), ctypes.c_uint32,
                                                    ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, _U16P,
                                                    ctypes.c_int32, _P]),
    "foil_matmul_tiles_gather_mc_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, _U16P, ctypes.c_uint32, ctypes.c_uint32,
                                                       ctypes.c_uint32, _U16P, ctypes.c_int32, _P]),
    "foil_matmul_tiles_gather_ce_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, ctypes.POINTER(_P), ctypes.c_uint32,
                                                       ctypes.c_uint32, ctypes.c_uint32, ctypes.c_uint32, _U16P,
                                                       ctypes.c_int32, ctypes.c_uint32, _P]),
    "foil_peer_alloc": (ctypes.c_int, [ctypes.c_int32, ctypes.c_uint64, ctypes.POINTER(_P),
                                       ctypes.POINTER(ctypes.c_uint8)]),
    "foil_peer_open": (ctypes.c_int, [ctypes.c_int32, ctypes.POINTER(ctypes.c_uint8), ctypes.POINTER(_P)]),
    "foil_peer_close": (ctypes.c_int, [ctypes.c_int32, _P]),
    "foil_peer_free": (ctypes.c_int, [ctypes.c_int32, _P]),
    "foil_set_wait_limit_ns": (ctypes.c_uint64, [ctypes.c_uint64]),
    "foil_conv2d_chw_dev": (ctypes.c_int, [_U16P, _U16P, _U16P, _U16P] + [ctypes.c_uint32] * 9 +
                            [ctypes.c_int32, _P]),
    "foil_w4_packed_bytes": (ctypes.c_uint64, [_U32, _U32, _U32, _I32]),
    "foil_w4_pack_dev": (ctypes.c_int, [_P, _U16P, _P, _P, _U32, _U32, _U32, _P]),
    "foil_w4_quantize_tiles_dev": (ctypes.c_int, [_U16P, _P, _U32, _U32, _U32, _I32, _P]),
    "foil_w4_dequantize_tiles_dev": (ctypes.c_int, [_P, _U16P, _U32, _U32, _U32, _I32, _I32, _P]),
    "foil_w4_matvec_dev": (ctypes.c_int, [_U16P, _U64, _P, _U16P, _U16P, _U64, _U32, _U32, _U32, _U32, _I32,
                                          _I32, _P]),
    "foil_block_norm_dev": (ctypes.c_int, [_P, _U64, _U16P, _U64, _I32, _U16P, _U16P, _U64, _U32, _I32, _U16P,
                                           _P, _U64, _U16P, _U64, _P, _P, _U32, _U32, _I32, _F32, _F32, _P]),
    "foil_block_norm_grad_ws_bytes": (ctypes.c_uint64, [_U32, _U32, _U32]),
    "foil_block_norm_grad_dev": (ctypes.c_int, [_P, _U64, _U16P, _U64, _P, _U64, _P, _U16P, _U16P, _U64, _I32,
                                                _P, _U16P, _U16P, _U64, _U32, _I32, _P, _U64, _U16P, _U64,
                                                _U16P, _U64, _P, _P, _P, _U64, _U32, _U32, _I32, _F32, _P]),
    "foil_embed_rows_dev": (ctypes.c_int, [_P, _I32, _U16P, _U64, _P, _U64, _U32, _U32, _U32, _I32, _F32,
                                           ctypes.c_int64, _P]),
    "foil_embed_rows_grad_ws_bytes": (ctypes.c_uint64, [_U32, _U32, _U32]),
    "foil_embed_rows_grad_dev": (ctypes.c_int, [_P, _I32, _P, _U64, _P, _U64, _U32, _U32, _U32, _I32, _F32,
                                                ctypes.c_int64, _I32, _P, _U64, _P]),
}

# Bits of the device error word (include/foil_c.h FOIL_DEVERR_*).
DEVERR_WAIT_TIMEOUT, DEVERR_BAD_SHAPE, DEVERR_CONFIG, DEVERR_BAD_INDEX = 1, 2, 4, 8

_lib = None


def lib():
    """Load lib/libfoil.so (raises if it has not been built)."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise FoilError(4, f"libfoil.so not built: {LIB_PATH} (run make -C tt-foil_b200)")
        L = ctypes.CDLL(LIB_PATH)
        for name, (res, args) in SIGNATURES.items():
            fn = getattr(L, name)
            fn.restype = res
            fn.argtypes = args
        _lib = L
    return _lib


def check(rc):
    if rc != FOIL_OK:
        msg = lib().foil_last_error().decode(errors="replace")
        raise FoilError(rc, msg)


def launch_count():
    return int(lib().foil_launch_count())


def set_wait_limit_ns(ns):
    """Wall-time limit of every bounded device-side wait for the launches
    that follow (0 = the default 2 s); returns the previous limit."""
    return int(lib().foil_set_wait_limit_ns(int(ns)))


# ------------------------------------------------------------ device layer ---

def _ptr(t):
    """Device pointer of a torch tensor or an int."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    return t.data_ptr()


_raw_stream = None


def _current_stream():
    """Handle of the current device's current stream.  torch's own short cut
    takes 0.1 us where the Stream object takes 3."""
    global _raw_stream
    if _raw_stream is None:
        import torch
        short = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if short is None:
            _raw_stream = lambda: torch.cuda.current_stream().cuda_stream  # noqa: E731
        else:
            _raw_stream = lambda: short(torch.cuda.current_device())  # noqa: E731
    return _raw_stream()


def _stream(stream):
    if stream is None:
        return _current_stream()
    if isinstance(stream, int):
        return stream
    return stream.cuda_stream


def tilize(row_major, tiles, rows, cols, stream=None):
    check(lib().foil_tilize_dev(_ptr(row_major), _ptr(tiles), rows, cols, _stream(stream)))


def untilize(tiles, row_major, rows, cols, stream=None):
    check(lib().foil_untilize_dev(_ptr(tiles), _ptr(row_major), rows, cols, _stream(stream)))


def tile_copy(src, dst, nbytes, stream=None):
    check(lib().foil_tile_copy_dev(_ptr(src), _ptr(dst), nbytes, _stream(stream)))


def add_tiles(a, b, out, n, stream=None):
    check(lib().foil_add_tiles_dev(_ptr(a), _ptr(b), _ptr(out), n, _stream(stream)))


def relu_tiles(x, out, n, stream=None):
    check(lib().foil_relu_tiles_dev(_ptr(x), _ptr(out), n, _stream(stream)))


def bias_add_tiles(x, bias_tiles, out, rows, cols, stream=None):
    check(lib().foil_bias_add_tiles_dev(_ptr(x), _ptr(bias_tiles), _ptr(out), rows, cols,
                                        _stream(stream)))


def matmul_tiles(a, b, c, Mt, Kt, Nt, bias=None, relu=False, stream=None):
    check(lib().foil_matmul_tiles_dev(_ptr(a), _ptr(b), _ptr(c), Mt, Kt, Nt, _ptr(bias),
                                      1 if relu else 0, _stream(stream)))


def matmul_tiles_gather(a, b, c, peer_c, Mt, Kt, Nt, bias=None, relu=False, stream=None):
    """matmul_tiles that also stores every output tile to the peer buffers
    `peer_c` (device addresses as ints, other GPUs' memory opened with
    peer_open, offset like c): C = A . B lands in c and in every peer copy."""
    arr = (_P * max(1, len(peer_c)))(*[int(x) for x in peer_c])
    check(lib().foil_matmul_tiles_gather_dev(_ptr(a), _ptr(b), _ptr(c), arr, len(peer_c), Mt, Kt, Nt,
                                             _ptr(bias), 1 if relu else 0, _stream(stream)))


def matmul_tiles_gather_mc(a, b, c, mc_c, Mt, Kt, Nt, bias=None, relu=False, stream=None):
    """matmul_tiles whose output tiles are stored through the NVLink
    multicast address `mc_c` (an int: c's offset in a multicast object bound
    on every GPU), so C lands in every GPU's copy."""
    check(lib().foil_matmul_tiles_gather_mc_dev(_ptr(a), _ptr(b), _ptr(c), _P(int(mc_c)), Mt, Kt, Nt, _ptr(bias),
                                                1 if relu else 0, _stream(stream)))


def matmul_tiles_gather_ce(a, b, c, peer_c, Mt, Kt, Nt, bias=None, relu=False, chunks=8, stream=None):
    """matmul_tiles_gather with the transfer on the copy engines: the GEMM
    runs in `chunks` row chunks and each finished chunk is copied to every
    peer buffer while the next one computes; `stream` continues after the
    last copy."""
    arr = (_P * max(1, len(peer_c)))(*[int(x) for x in peer_c])
    check(lib().foil_matmul_tiles_gather_ce_dev(_ptr(a), _ptr(b), _ptr(c), arr, len(peer_c), Mt, Kt, Nt,
                                                _ptr(bias), 1 if relu else 0, int(chunks), _stream(stream)))


PEER_HANDLE_BYTES = 64


def peer_alloc(device, nbytes):
    """Device buffer on CUDA device `device` shareable with the node's other
    processes: returns (device address, 64-byte export handle)."""
    ptr = _P()
    h = (ctypes.c_uint8 * PEER_HANDLE_BYTES)()
    check(lib().foil_peer_alloc(device, nbytes, ctypes.byref(ptr), h))
    return int(ptr.value), bytes(h)


def peer_open(device, handle):
    """Open another process's peer_alloc buffer on CUDA device `device`;
    returns its device address there."""
    if len(handle) != PEER_HANDLE_BYTES:
        raise FoilError(1, "peer_open: handle must be 64 bytes")
    ptr = _P()
    h = (ctypes.c_uint8 * PEER_HANDLE_BYTES).from_buffer_copy(handle)
    check(lib().foil_peer_open(device, h, ctypes.byref(ptr)))
    return int(ptr.value)


def peer_close(device, ptr):
    check(lib().foil_peer_close(device, ptr))


def peer_free(device, ptr):
    check(lib().foil_peer_free(device, ptr))


def conv2d_nhwc(x, w, bias, y, N, H, W, Cin, Cout, KH, KW, stride, pad, relu=False, stream=None):
    """y (N,Ho,Wo,Cout) = relu?(conv(x (N,H,W,Cin), w (Cout,KH,KW,Cin)) + bias)."""
    check(lib().foil_conv2d_nhwc_dev(_ptr(x), _ptr(w), _ptr(bias), _ptr(y), N, H, W, Cin, Cout, KH,
                                     KW, stride, pad, 1 if relu else 0, _stream(stream)))


def conv2d_chw(x, w, bias, y, N, Cin, H, W, Cout, KH, KW, stride, pad, relu=False, stream=None):
    """The reference's convention: y (N,Cout,Ho,Wo) = relu?(conv(x (N,Cin,H,W),
    w (Cout, Cin*KH*KW)) + bias), operands re-laid on the device."""
    check(lib().foil_conv2d_chw_dev(_ptr(x), _ptr(w), _ptr(bias), _ptr(y), N, Cin, H, W, Cout, KH, KW, stride,
                                    pad, 1 if relu else 0, _stream(stream)))


# ------------------------------------------------------ token-path operators ---

# Their kernels take a few microseconds, so the calls below look at a tensor as
# little as they can.

def _place(stream):
    """The current device, and the handle of `stream` or of its current stream."""
    global _place_of
    if _place_of is None:
        import torch
        torch.cuda.current_device()  # sets CUDA up; from then on torch's own short cut does
        _place_of = (getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device),
                     getattr(torch._C, "_cuda_getCurrentRawStream", None))
    device = _place_of[0]()
    if stream is None and _place_of[1] is not None:
        return device, _place_of[1](device)
    return device, _stream(stream)


_place_of = None


# What a tensor's elements may be: the kind's own type, which the calls below look
# for first, others that stand for it, and its name.
class _Kind:
    def __init__(self, name, *types):
        self.name, self.types, self.own = name, types, None

    def check(self, t):
        if self.own is None:
            import torch
            self.types = tuple(getattr(torch, n) for n in self.types if hasattr(torch, n))
            self.own = self.types[0]
        if t.dtype not in self.types:
            raise FoilError(1, f"tt-foil: a tensor is {t.dtype}, not {self.name}")


_BF16 = _Kind("bf16 (or 16-bit integers)", "bfloat16", "int16", "uint16")
_FP32 = _Kind("float32", "float32")
_BYTES = _Kind("bytes", "uint8", "int8")
_IDS = _Kind("32- or 64-bit integers", "int64", "int32", "uint32", "uint64")


def _vec(t, device, kind=None, n=0):
    """Pointer of a dense argument of at least `n` elements: a torch tensor on
    `device`, an address or None."""
    if t is None:
        return None
    try:
        if t.get_device() != device:
            raise FoilError(1, "tt-foil: a tensor is not on the current CUDA device")
    except AttributeError:
        return t  # an address
    if not t.is_contiguous():
        raise FoilError(1, "tt-foil: a tensor must be contiguous")
    if kind is not None and t.dtype is not kind.own:
        kind.check(t)
    if t.numel() < n:
        raise FoilError(1, f"tt-foil: a tensor has {t.numel()} elements, {n} are needed")
    return t.data_ptr()


def _mat(t, ld, device, cols=None, rows=0, kind=None):
    """Pointer and row stride in elements of a matrix of `rows` x `cols`: the
    stride as given, else that of a 2-D torch tensor, else 0 (dense)."""
    if t is None:
        return None, ld
    try:
        if t.get_device() != device:
            raise FoilError(1, "tt-foil: a tensor is not on the current CUDA device")
    except AttributeError:
        return t, ld  # an address
    if kind is not None and t.dtype is not kind.own:
        kind.check(t)
    if not ld and t.shape == (rows, cols) and t.is_contiguous():
        return t.data_ptr(), 0
    return t.data_ptr(), _stride(t, ld, cols, rows)


def _stride(t, ld, cols, rows):
    """A tensor's row stride in elements where it is not `rows` dense rows of `cols`."""
    if ld:
        if rows and t.storage_offset() + (rows - 1) * ld + cols > t.untyped_storage().nbytes() // t.element_size():
            raise FoilError(1, f"tt-foil: {rows} x {cols} values with a row stride of {ld} pass a tensor's end")
        return ld
    shape = t.shape
    dims = len(shape)
    if t.is_contiguous() and (shape[1] == cols if dims == 2 else dims < 2 or not rows or shape[-1] == cols):
        if rows and t.numel() < rows * cols:
            raise FoilError(1, f"tt-foil: a tensor has {t.numel()} elements, {rows} x {cols} are needed")
        return 0
    if dims != 2:
        raise FoilError(1, "tt-foil: a tensor must be contiguous rows, or a matrix with a row stride")
    if rows and (shape[0] < rows or shape[1] < cols):
        raise FoilError(1, f"tt-foil: a tensor is {shape[0]} x {shape[1]}, {rows} x {cols} are needed")
    rows, cols = shape
    step, unit = t.stride()
    if (cols > 1 and unit != 1) or (rows > 1 and step < cols):
        raise FoilError(1, "tt-foil: rows of a tensor must be contiguous and must not overlap")
    return step if rows > 1 else 0


def _is_fp32(fp32, *tensors):
    """The residual stream's type: as given, else from the first torch tensor (float32 or bf16)."""
    for t in tensors:
        if not (t is None or isinstance(t, int)):
            own = t.dtype
            wide = own is _FP32.own
            if not wide and own is not _BF16.own:
                wide = t.element_size() == 4
                (_FP32 if wide else _BF16).check(t)
            if fp32 is not None and bool(fp32) is not wide:
                raise FoilError(1, "tt-foil: tensors of one type are mixed with another")
            fp32 = wide
    return 1 if fp32 else 0


def w4_packed_bytes(K, N, group, zeros=False):
    """Bytes of the 4-bit storage of a K x N weight matrix (0: sizes out of range)."""
    return int(lib().foil_w4_packed_bytes(K, N, group, 1 if zeros else 0))


# Bytes of a storage block, by (group, zero points); 0 for groups that the call refuses.
_BLOCK_BYTES = {(g, z): 1024 + (6144 if z else 4096) // g for g in (32, 64, 128) for z in (False, True)}


def _packed(t, device, K, N, group, zeros):
    """Pointer of 4-bit storage (the size of w4_packed_bytes)."""
    return _vec(t, device, _BYTES, (N + 15 >> 4) * (K + 127 >> 7) * _BLOCK_BYTES.get((group, not not zeros), 0))


def _tiles(t, device, rows, cols):
    """Pointer of a tile stream of rows x cols tiles."""
    return _vec(t, device, _BF16, rows * cols * 1024)


def w4_pack(codes, scales, packed, K, N, group, zero_points=None, stream=None):
    """Codes (N x K, one byte each), scales (N x ceil(K / group) bf16) and zero
    points (alike, one byte each, or None) -> 4-bit storage."""
    dev, stream = _place(stream)
    groups = N * -(-K // group) if group > 0 else 0
    rc = (_lib or lib()).foil_w4_pack_dev(
        _vec(codes, dev, _BYTES, N * K), _vec(scales, dev, _BF16, groups), _vec(zero_points, dev, _BYTES, groups),
        _packed(packed, dev, K, N, group, zero_points is not None), K, N, group, stream)
    if rc:
        check(rc)


def w4_quantize_tiles(tiles, packed, Kt, Nt, group, zeros=False, stream=None):
    """Tile stream of Kt x Nt tiles -> 4-bit storage with a scale (and, with
    `zeros`, a zero point) for each `group` values of a column."""
    dev, stream = _place(stream)
    rc = (_lib or lib()).foil_w4_quantize_tiles_dev(
        _tiles(tiles, dev, Kt, Nt), _packed(packed, dev, 32 * Kt, 32 * Nt, group, zeros), Kt, Nt, group,
        1 if zeros else 0, stream)
    if rc:
        check(rc)


def w4_dequantize_tiles(packed, tiles, K, N, group, zeros=False, transpose=False, stream=None):
    """4-bit storage -> tile stream of the weights, or of their transpose."""
    dev, stream = _place(stream)
    rc = (_lib or lib()).foil_w4_dequantize_tiles_dev(
        _packed(packed, dev, K, N, group, zeros), _tiles(tiles, dev, -(-K // 32), -(-N // 32)), K, N, group,
        1 if zeros else 0, 1 if transpose else 0, stream)
    if rc:
        check(rc)


def w4_matvec(x, packed, y, M, K, N, group, zeros=False, bias=None, relu=False, ld_x=0, ld_y=0, stream=None):
    """y (M x N) = relu?(x (M x K) . W + bias) with 4-bit W, M at most 64."""
    dev, stream = _place(stream)
    x, ld_x = _mat(x, ld_x, dev, K, M, _BF16)
    y, ld_y = _mat(y, ld_y, dev, N, M, _BF16)
    rc = (_lib or lib()).foil_w4_matvec_dev(
        x, ld_x, _packed(packed, dev, K, N, group, zeros), _vec(bias, dev, _BF16, N), y, ld_y, M, K, N, group,
        1 if zeros else 0, 1 if relu else 0, stream)
    if rc:
        check(rc)


GATE_ACTS = {"none": 0, "sigmoid": 1}


def _gate_act(name):
    if name not in GATE_ACTS:
        raise FoilError(1, f"tt-foil: unknown gate activation {name!r}")
    return GATE_ACTS[name]


def _gates(T, gate_rows):
    """Gate rows of T tokens."""
    return T if gate_rows == 1 else -(-T // gate_rows) if gate_rows > 0 else 0


def block_norm(resid, u, h, y, T, D, w_pre=None, post=False, w_post=None, gate=None, gate_rows=1, gate_act="none",
               scale=1.0, eps=1e-5, rstd_post=None, rstd_pre=None, fp32=None, ld_resid=0, ld_u=0, ld_gate=0, ld_h=0,
               ld_y=0, stream=None):
    """h = resid + scale * act(gate) * (post ? N(u) * w_post : u);
    y = N(h) * w_pre, with N(v) = v / sqrt(mean(v^2) + eps).  resid and h are
    bf16 or fp32 (taken from the tensors; `fp32` for raw pointers)."""
    dev, stream = _place(stream)
    wide = _is_fp32(fp32, resid, h)
    resid, ld_resid = _mat(resid, ld_resid, dev, D, T)
    u, ld_u = _mat(u, ld_u, dev, D, T, _BF16)
    if gate is not None:
        gate, ld_gate = _mat(gate, ld_gate, dev, D, _gates(T, gate_rows), _BF16)
    h, ld_h = _mat(h, ld_h, dev, D, T)
    y, ld_y = _mat(y, ld_y, dev, D, T, _BF16)
    rc = (_lib or lib()).foil_block_norm_dev(
        resid, ld_resid, u, ld_u, 1 if post else 0, _vec(w_post, dev, _BF16, D), gate, ld_gate, gate_rows,
        _gate_act(gate_act), _vec(w_pre, dev, _BF16, D), h, ld_h, y, ld_y, _vec(rstd_post, dev, _FP32, T),
        _vec(rstd_pre, dev, _FP32, T), T, D, wide, scale, eps, stream)
    if rc:
        check(rc)


def block_norm_grad_ws_bytes(T, D, gate_rows=0):
    """Workspace bytes of block_norm_grad (gate_rows 0: no gate)."""
    return int(lib().foil_block_norm_grad_ws_bytes(T, D, gate_rows))


def block_norm_grad(dh, dy, h, u, dresid, du, T, D, ws, rstd_pre=None, w_pre=None, dw_pre=None, post=False,
                    rstd_post=None, w_post=None, dw_post=None, gate=None, dgate=None, gate_rows=1, gate_act="none",
                    scale=1.0, fp32=None, ws_bytes=None, ld_dh=0, ld_dy=0, ld_h=0, ld_u=0, ld_gate=0, ld_dresid=0,
                    ld_du=0, ld_dgate=0, stream=None):
    """Gradients of block_norm from those of h (dh) and y (dy); outputs that
    are None are not made.  `ws`: a workspace of block_norm_grad_ws_bytes."""
    dev, stream = _place(stream)
    wide = _is_fp32(fp32, dh, h, dresid)
    n = _ws_bytes(ws, ws_bytes)
    dh, ld_dh = _mat(dh, ld_dh, dev, D, T)
    dy, ld_dy = _mat(dy, ld_dy, dev, D, T, _BF16)
    h, ld_h = _mat(h, ld_h, dev, D, T)
    u, ld_u = _mat(u, ld_u, dev, D, T, _BF16)
    dresid, ld_dresid = _mat(dresid, ld_dresid, dev, D, T)
    du, ld_du = _mat(du, ld_du, dev, D, T, _BF16)
    if gate is not None:
        gates = _gates(T, gate_rows)
        gate, ld_gate = _mat(gate, ld_gate, dev, D, gates, _BF16)
        dgate, ld_dgate = _mat(dgate, ld_dgate, dev, D, gates, _BF16)
    elif dgate is not None:
        dgate, ld_dgate = _mat(dgate, ld_dgate, dev, D)
    rc = (_lib or lib()).foil_block_norm_grad_dev(
        dh, ld_dh, dy, ld_dy, h, ld_h, _vec(rstd_pre, dev, _FP32, T), _vec(w_pre, dev, _BF16, D), u, ld_u,
        1 if post else 0, _vec(rstd_post, dev, _FP32, T), _vec(w_post, dev, _BF16, D), gate, ld_gate, gate_rows,
        _gate_act(gate_act), dresid, ld_dresid, du, ld_du, dgate, ld_dgate, _vec(dw_post, dev, _FP32, D),
        _vec(dw_pre, dev, _FP32, D), _vec(ws, dev), n, T, D, wide, scale, stream)
    if rc:
        check(rc)


def _ws_bytes(ws, ws_bytes):
    if ws is None or isinstance(ws, int):
        return ws_bytes or 0
    n = ws.numel() * ws.element_size()
    if ws_bytes is not None and ws_bytes > n:
        raise FoilError(1, f"tt-foil: the workspace has {n} bytes, not {ws_bytes}")
    return n if ws_bytes is None else ws_bytes


def _id_bytes(ids, id_bytes):
    if isinstance(ids, int) or ids is None:
        return id_bytes
    if ids.dtype is not _IDS.own:
        _IDS.check(ids)
    return ids.element_size()


def embed_rows(ids, table, out, T, V, D, scale=1.0, pad_id=-1, id_bytes=4, fp32=None, ld_table=0, ld_out=0,
               stream=None):
    """out[t] = scale * table[ids[t]]; zeros where ids[t] is pad_id.  A bad id
    gives zeros and DEVERR_BAD_INDEX (see device_error)."""
    dev, stream = _place(stream)
    id_bytes, wide = _id_bytes(ids, id_bytes), _is_fp32(fp32, out)
    table, ld_table = _mat(table, ld_table, dev, D, V, _BF16)
    out, ld_out = _mat(out, ld_out, dev, D, T)
    rc = (_lib or lib()).foil_embed_rows_dev(
        _vec(ids, dev, None, T), id_bytes, table, ld_table, out, ld_out, T, V, D, wide, scale, pad_id, stream)
    if rc:
        check(rc)


def embed_rows_grad_ws_bytes(T, V, D):
    """Workspace bytes of embed_rows_grad."""
    return int(lib().foil_embed_rows_grad_ws_bytes(T, V, D))


def embed_rows_grad(ids, dout, dtable, T, V, D, ws, scale=1.0, pad_id=-1, accumulate=False, id_bytes=4, fp32=None,
                    ws_bytes=None, ld_dout=0, ld_dtable=0, stream=None):
    """dtable[v] (fp32) = scale * sum of dout[t] over ids[t] = v, or with
    `accumulate` added to what is there.  `ws`: a workspace of
    embed_rows_grad_ws_bytes."""
    dev, stream = _place(stream)
    id_bytes, wide, n = _id_bytes(ids, id_bytes), _is_fp32(fp32, dout), _ws_bytes(ws, ws_bytes)
    dout, ld_dout = _mat(dout, ld_dout, dev, D, T)
    dtable, ld_dtable = _mat(dtable, ld_dtable, dev, D, V, _FP32)
    rc = (_lib or lib()).foil_embed_rows_grad_dev(
        _vec(ids, dev, None, T), id_bytes, dout, ld_dout, dtable, ld_dtable, T, V, D, wide, scale, pad_id,
        1 if accumulate else 0, _vec(ws, dev), n, stream)
    if rc:
        check(rc)


def matmul_tiles_host(device, a, b, c, Mt, Kt, Nt, bias=None, relu=False, chunk_rows=0):
    """Pipelined C = A . B (+bias, relu) on host tile streams (pinned CPU
    tensors, numpy arrays or host addresses): copies, GEMM chunks and
    read-back overlap; returns when C is in host memory."""
    check(lib().foil_matmul_tiles_host(device, _hptr(a), _hptr(b), _hptr(c), Mt, Kt, Nt, _hptr(bias),
                                       1 if relu else 0, chunk_rows))


def conv2d_nhwc_host(device, x, w, bias, y, N, H, W, Cin, Cout, KH, KW, stride, pad, relu=False,
                     chunk_images=0):
    """Pipelined NHWC convolution on host buffers (see matmul_tiles_host)."""
    check(lib().foil_conv2d_nhwc_host(device, _hptr(x), _hptr(w), _hptr(bias), _hptr(y), N, H, W, Cin,
                                      Cout, KH, KW, stride, pad, 1 if relu else 0, chunk_images))


def host_pipeline_release(device):
    check(lib().foil_host_pipeline_release(device))


def _hptr(t):
    """Host address of a CPU torch tensor, a numpy array or an int (None -> NULL)."""
    if t is None:
        return None
    if isinstance(t, int):
        return t
    if hasattr(t, "ctypes"):
        return t.ctypes.data
    assert not t.is_cuda, "host pipeline entry points take host memory"
    return t.data_ptr()


def device_error(stream=None):
    """Read and clear the device-side error word (synchronizes the stream)."""
    v = ctypes.c_uint32(0)
    check(lib().foil_device_error_dev(_stream(stream), ctypes.byref(v)))
    return v.value


# ----------------------------------------------------------- runtime layer ---

class Buffer:
    def __init__(self, c):
        self.c = c

    @property
    def device_addr(self):
        return int(self.c.device_addr)

    @property
    def size_bytes(self):
        return int(self.c.size_bytes)


class Kernel:
    def __init__(self, device, handle):
        self.device = device
        self.handle = handle

    def __del__(self):
        if self.handle and _lib is not None:
            _lib.foil_release_kernel(self.handle)
            self.handle = None


class Device:
    """tt-foil device (open_device ... close_device) over the C-ABI."""

    def __init__(self, index=0, cores=((0, 0),), firmware_dir=""):
        arr = (foil_core * len(cores))(*[foil_core(x, y) for x, y in cores])
        h = ctypes.c_void_p()
        check(lib().foil_open_device(index, firmware_dir.encode(), arr, len(cores), ctypes.byref(h)))
        self.handle = h

    def close(self):
        if self.handle:
            h, self.handle = self.handle, None
            check(lib().foil_close_device(h))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def allocate(self, loc, size, core=(0, 0)):
        b = foil_buffer()
        check(lib().foil_allocate_buffer(self.handle, loc, size, foil_core(*core), ctypes.byref(b)))
        return Buffer(b)

    def write(self, buf, src_ptr, nbytes):
        check(lib().foil_write_buffer(self.handle, ctypes.byref(buf.c), src_ptr, nbytes))

    def read(self, buf, dst_ptr, nbytes):
        check(lib().foil_read_buffer(self.handle, ctypes.byref(buf.c), dst_ptr, nbytes))

    def write_array(self, buf, arr):
        import numpy as np
        a = np.ascontiguousarray(arr)
        self.write(buf, a.ctypes.data, a.nbytes)

    def read_array(self, buf, dtype, count):
        import numpy as np
        a = np.empty(count, dtype=dtype)
        self.read(buf, a.ctypes.data, a.nbytes)
        return a

    def device_ptr(self, buf):
        p = ctypes.c_void_p()
        check(lib().foil_buffer_device_ptr(self.handle, ctypes.byref(buf.c), ctypes.byref(p)))
        return int(p.value)

    def load_kernel(self, binaries, core=(0, 0)):
        keep = [(r, p.encode()) for r, p in binaries]
        arr = (foil_risc_binary * len(keep))(*[foil_risc_binary(r, p) for r, p in keep])
        h = ctypes.c_void_p()
        check(lib().foil_load_kernel(self.handle, arr, len(keep), foil_core(*core), ctypes.byref(h)))
        return Kernel(self, h)

    def load_program(self, program, core=(0, 0), reader="reader.brisc.elf"):
        """Load the standard five descriptors of programs/<program>/."""
        d = os.path.join(PROGRAMS_DIR, program)
        bins = [(BRISC, os.path.join(d, reader)), (NCRISC, os.path.join(d, "writer.ncrisc.elf")),
                (TRISC0, os.path.join(d, "compute.trisc0.elf")),
                (TRISC1, os.path.join(d, "compute.trisc1.elf")),
                (TRISC2, os.path.join(d, "compute.trisc2.elf"))]
        return self.load_kernel(bins, core)

    def set_runtime_args(self, kernel, risc, args):
        arr = (ctypes.c_uint32 * len(args))(*[int(a) & 0xffffffff for a in args])
        check(lib().foil_set_runtime_args(self.handle, kernel.handle, risc, arr, len(args)))

    def register_cbs(self, kernel, cbs):
        arr = (foil_cb_config * len(cbs))(*[foil_cb_config(*c) for c in cbs])
        check(lib().foil_register_cbs(self.handle, kernel.handle, arr, len(cbs)))

    def execute(self, kernels, timeout_ms=5000):
        if not isinstance(kernels, (list, tuple)):
            kernels = [kernels]
        arr = (ctypes.c_void_p * len(kernels))(*[k.handle for k in kernels])
        check(lib().foil_execute(self.handle, arr, len(kernels), timeout_ms))

    def noc_unicast_addr(self, core, l1_addr):
        out = ctypes.c_uint64()
        check(lib().foil_make_noc_unicast_addr(self.handle, foil_core(*core), l1_addr, ctypes.byref(out)))
        return int(out.value)

    def noc_dram_addr(self, offset):
        out = ctypes.c_uint64()
        check(lib().foil_make_noc_dram_addr(self.handle, offset, ctypes.byref(out)))
        return int(out.value)


def lo(v):
    return v & 0xffffffff


def hi(v):
    return (v >> 32) & 0xffffffff
