"""ctypes binding of the C++ MoE layer engine (include/gyro_moe.h) and its operators (include/gyro_ops.h)."""
from __future__ import annotations

import ctypes as C
import struct
import sys

import numpy as np

from . import BUILD_DIR, KERNEL_DIR

LIB_PATH = BUILD_DIR / "libgyro_moe.so"
PATH_REFERENCE, PATH_DECODE, PATH_PREFILL, PATH_GENERIC = 0, 1, 2, 3


class LayerDesc(C.Structure):
    _fields_ = [("E", C.c_uint32), ("F", C.c_uint32), ("n_expert", C.c_uint32), ("n_used", C.c_uint32),
                ("expert_weights_scale", C.c_float),
                ("router", C.c_void_p), ("router_bias", C.c_void_p), ("gate_signs", C.c_void_p),
                ("down_signs", C.c_void_p), ("gate", C.c_void_p), ("up", C.c_void_p), ("down", C.c_void_p),
                ("types", C.c_void_p), ("SF", C.c_uint32), ("sh_gate", C.c_void_p), ("sh_up", C.c_void_p),
                ("sh_down", C.c_void_p), ("sh_gate_inp", C.c_void_p), ("norm_weight", C.c_void_p),
                ("norm_eps", C.c_float), ("sh_type", C.c_uint32)]


class Rows(C.Structure):
    _fields_ = [("data", C.c_void_p), ("stride", C.c_uint64), ("type", C.c_uint32), ("reserved", C.c_uint32)]


class MatrixDesc(C.Structure):
    _fields_ = [("format", C.c_uint32), ("rows", C.c_uint32), ("cols", C.c_uint32), ("group", C.c_uint32)] + \
        [(p + f, C.c_void_p) for p in ("", "up_") for f in ("quants", "scales", "mins")]


class BlockNormDesc(C.Structure):
    _fields_ = [("E", C.c_uint32), ("post", C.c_uint32), ("gate_kind", C.c_uint32), ("gate_act", C.c_uint32),
                ("h", Rows), ("x", Rows), ("out", Rows), ("normed", Rows), ("gate", Rows),
                ("post_weight", C.c_void_p), ("pre_weight", C.c_void_p), ("post_eps", C.c_float),
                ("pre_eps", C.c_float), ("scale", C.c_float), ("reserved", C.c_uint32)]


class LogprobsDesc(C.Structure):
    _fields_ = [("logits", Rows), ("V", C.c_uint32), ("given", C.c_uint32), ("top", C.c_uint32),
                ("tokens_64", C.c_uint32), ("scale", C.c_float), ("reserved", C.c_uint32), ("tokens", C.c_void_p),
                ("tokens_stride", C.c_uint64), ("logprobs", C.c_void_p), ("logprobs_stride", C.c_uint64),
                ("entropy", C.c_void_p), ("top_ids", C.c_void_p), ("top_logprobs", C.c_void_p),
                ("top_stride", C.c_uint64), ("workspace", C.c_void_p), ("workspace_bytes", C.c_uint64)]


# 4-bit matrix formats (gm_matrix_desc) and the operators' activations and element types.
MATRIX_FORMATS = {"q4_0": 0, "q4_1": 1, "q4": 2}
ACTS = {"none": 0, "silu": 1, "sigmoid": 2}
GATE_TOKEN, GATE_CHANNEL, GATE_VALUE = 1, 2, 3
_TYPE_NAMES = {"torch.float32": 0, "torch.bfloat16": 1, "torch.float16": 2, "torch.int32": 3, "torch.int64": 4,
               "torch.uint8": 5}
_type_codes = {}  # dtype object -> its code in _TYPE_NAMES
_ROW_TYPES, _FLOAT, _INT32, _INTS, _UINT8 = (0, 1, 2), (0,), (3,), (3, 4), (5,)

# The structs above as bytes, which ctypes passes several times faster than it fills a Structure.
_PACK_ROWS = struct.Struct("@PQII").pack
_PACK_NORM = struct.Struct("@4I" + 5 * "PQII" + "PP4f").pack
_PACK_LOGPROBS = struct.Struct("@PQII4IfIPQPQPPPQPQ").pack
_NO_ROWS = (0, 0, 0)


def _count(n, what):
    """n, which the library takes in 32 bits (ctypes would drop the rest)."""
    if not 0 <= n <= 0xffffffff:
        raise ValueError(f"{what}: {n} is not a 32-bit count")
    return n


def _type(t, allowed, what):
    code = _type_codes.get(t.dtype)
    if code is None:
        code = _type_codes[t.dtype] = _TYPE_NAMES.get(str(t.dtype), -1)
    if code not in allowed:
        raise ValueError(f"{what}: dtype {t.dtype} is not taken")
    return code


# GGML type of a shared expert's matrices (src/kernels.zig:7-10) -> the engine's gm_layer_desc code.
SHARED_KIND = {30: 0, 8: 1, 0: 2}


_lib = None


def lib() -> C.CDLL:
    global _lib
    if _lib is None:
        if not LIB_PATH.exists():
            raise RuntimeError(f"{LIB_PATH} is not built; run gyro-dx_amd/build.py")
        L = C.CDLL(str(LIB_PATH))
        vp, u32, f32p = C.c_void_p, C.c_uint32, C.POINTER(C.c_float)
        L.gm_create.argtypes = [C.c_char_p, u32, u32, C.POINTER(vp)]
        L.gm_destroy.argtypes = [vp]
        L.gm_destroy.restype = None
        L.gm_last_error.argtypes = [vp]
        L.gm_last_error.restype = C.c_char_p
        L.gm_add_layer.argtypes = [vp, C.POINTER(LayerDesc), C.POINTER(u32)]
        L.gm_forward.argtypes = [vp, u32, u32, f32p, u32, f32p]
        L.gm_last_routes.argtypes = [vp, u32, C.POINTER(u32), f32p]
        L.gm_last_sort.argtypes = [vp, u32, C.POINTER(u32), C.POINTER(u32)]
        L.gm_dequant.argtypes = [vp, u32, u32, u32, u32, u32, f32p]
        L.gm_dequant_as.argtypes = [vp, u32, u32, u32, u32, u32, u32, f32p]
        L.gm_set_tokens.argtypes = [vp, f32p, u32]
        L.gm_run.argtypes = [vp, u32, u32, u32, u32, C.POINTER(u32), u32, C.POINTER(C.c_double),
                             C.POINTER(C.c_double)]
        L.gm_run_bracketed.argtypes = [vp, u32, u32, u32, u32, C.POINTER(u32), u32, u32, C.POINTER(C.c_double),
                                       C.POINTER(C.c_double), C.POINTER(C.c_double)]
        L.gm_read_outputs.argtypes = [vp, f32p, u32]
        L.gm_last_tiles.argtypes = [vp, u32, C.POINTER(u32), C.POINTER(u32)]
        L.gm_forward_stack.argtypes = [vp, C.POINTER(u32), u32, u32, f32p, u32, f32p]
        L.gm_run_stack.argtypes = [vp, u32, u32, u32, u32, C.POINTER(u32), u32, C.POINTER(C.c_double),
                                   C.POINTER(C.c_double)]
        L.gm_forward_decode_noalloc.argtypes = [vp, u32, vp, u32, vp, vp]
        L.gm_load_operators.argtypes = [vp]
        L.gm_add_matrix.argtypes = [vp, C.POINTER(MatrixDesc), C.POINTER(u32)]
        L.gm_release_matrix.argtypes = [vp, u32]
        L.gm_linear.argtypes = [vp, u32, vp, u32, vp, u32, u32, C.c_float, vp]
        L.gm_block_norm.argtypes = [vp, vp, u32, vp]
        L.gm_logprobs_workspace.argtypes = [u32, u32, u32]
        L.gm_logprobs_workspace.restype = C.c_uint64
        L.gm_logprobs.argtypes = [vp, vp, u32, vp]
        _lib = L
    return _lib


def _f32p(a):
    return a.ctypes.data_as(C.POINTER(C.c_float))


class Engine:
    """The MoE layer engine on one GPU. Layers come from gyrodx.synth.Layer objects."""

    def __init__(self, max_tok: int = 64, adapter: int = 0, kernel_dir=KERNEL_DIR):
        self._h = C.c_void_p()
        rc = lib().gm_create(str(kernel_dir).encode(), adapter, max_tok, C.byref(self._h))
        if rc != 0:
            raise RuntimeError(f"gm_create failed ({rc})")
        self.max_tok = max_tok
        self.adapter = adapter
        self.E = None
        self._matrices = {}

    def _check(self, rc, what):
        if rc != 0:
            raise RuntimeError(f"{what} failed ({rc}): {lib().gm_last_error(self._h).decode()}")

    def close(self):
        if self._h:
            lib().gm_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

    def add_layer(self, layer) -> int:
        keep = []

        def ptr(a):
            if a is None:
                return None
            a = np.ascontiguousarray(a)
            keep.append(a)
            return a.ctypes.data

        def ptrs(mats):
            arr = (C.c_void_p * len(mats))(*[ptr(m) for m in mats])
            keep.append(arr)
            return C.cast(arr, C.c_void_p).value

        d = LayerDesc(E=layer.E, F=layer.F, n_expert=layer.n_expert, n_used=layer.n_used,
                      expert_weights_scale=layer.expert_weights_scale,
                      router=ptr(np.asarray(layer.router, np.float32)),
                      router_bias=ptr(None if layer.router_bias is None else np.asarray(layer.router_bias, np.float32)),
                      gate_signs=ptr(layer.gate_signs), down_signs=ptr(layer.down_signs),
                      gate=ptrs(layer.gate), up=ptrs(layer.up), down=ptrs(layer.down),
                      types=ptr(np.ascontiguousarray(layer.types, np.uint32).reshape(-1)),
                      SF=layer.SF, sh_gate=ptr(layer.sh_gate), sh_up=ptr(layer.sh_up), sh_down=ptr(layer.sh_down),
                      sh_gate_inp=ptr(None if layer.sh_gate_inp is None else np.asarray(layer.sh_gate_inp, np.float32)),
                      norm_weight=ptr(None if layer.norm_weight is None else np.asarray(layer.norm_weight, np.float32)),
                      norm_eps=layer.norm_eps, sh_type=SHARED_KIND[getattr(layer, "sh_type", 30)] if layer.SF else 0)
        idx = C.c_uint32()
        self._check(lib().gm_add_layer(self._h, C.byref(d), C.byref(idx)), "gm_add_layer")
        self.E, self.U, self.n_expert = layer.E, layer.n_used, layer.n_expert
        return idx.value

    def forward(self, layer: int, x: np.ndarray, path: int = PATH_DECODE) -> np.ndarray:
        x = np.ascontiguousarray(x, np.float32)
        out = np.empty_like(x)
        self._check(lib().gm_forward(self._h, layer, path, _f32p(x), x.shape[0], _f32p(out)), "gm_forward")
        return out

    def last_routes(self, n: int):
        ids = np.empty((n, self.U), np.uint32)
        w = np.empty((n, self.U), np.float32)
        self._check(lib().gm_last_routes(self._h, n, ids.ctypes.data_as(C.POINTER(C.c_uint32)), _f32p(w)),
                    "gm_last_routes")
        return ids, w

    def last_sort(self, n: int):
        """Counting sort of the last prefill forward: (route_order[n * n_used], order_start[n_expert + 1])."""
        order = np.empty(n * self.U, np.uint32)
        start = np.empty(self.n_expert + 1, np.uint32)
        p = lambda a: a.ctypes.data_as(C.POINTER(C.c_uint32))
        self._check(lib().gm_last_sort(self._h, n, p(order), p(start)), "gm_last_sort")
        return order, start

    def dequant(self, layer: int, expert: int, proj: int, row0: int, rows: int, cols: int,
                decoder: int = 0) -> np.ndarray:
        """Rows of one expert projection through a path's device decoder: 0 the decode kernels',
        1 the prefill GEMMs' (fp32 scale x codebook), 2 the prefill B operand (binary16)."""
        out = np.empty((rows, cols), np.float32)
        self._check(lib().gm_dequant_as(self._h, layer, expert, proj, row0, rows, decoder, _f32p(out)), "gm_dequant_as")
        return out

    def set_tokens(self, x: np.ndarray):
        x = np.ascontiguousarray(x, np.float32)
        self._check(lib().gm_set_tokens(self._h, _f32p(x), x.shape[0]), "gm_set_tokens")
        self.n_tokens = x.shape[0]

    def run(self, path: int, batch: int, calls: int, layers, bracket: int = 0, first: int = 0):
        """Processes `calls` calls of `batch` device-resident tokens from token `first`; returns
        (device ms, wall ms, mean duration in us of the bracketed kernel's launches)."""
        arr = (C.c_uint32 * len(layers))(*layers)
        dev, wall, br = C.c_double(), C.c_double(), C.c_double()
        self._check(lib().gm_run_bracketed(self._h, path, batch, calls, first, arr, len(layers), bracket,
                                           C.byref(dev), C.byref(wall), C.byref(br)), "gm_run")
        return dev.value, wall.value, br.value

    def last_tiles(self, max_tiles: int = 4096) -> np.ndarray:
        """Tile list of the last prefill call: [count, 4] u32 {expert, first row, rows, 0}."""
        buf = np.zeros((max_tiles, 4), np.uint32)
        cnt = C.c_uint32()
        self._check(lib().gm_last_tiles(self._h, max_tiles, buf.ctypes.data_as(C.POINTER(C.c_uint32)), C.byref(cnt)),
                    "gm_last_tiles")
        return buf[:cnt.value].copy()

    def forward_stack(self, layers, x: np.ndarray, path: int = PATH_DECODE) -> np.ndarray:
        """x <- x + MoE_l(RMSNorm_l(x)) over the given layer indices."""
        x = np.ascontiguousarray(x, np.float32)
        out = np.empty_like(x)
        arr = (C.c_uint32 * len(layers))(*layers)
        self._check(lib().gm_forward_stack(self._h, arr, len(layers), path, _f32p(x), x.shape[0], _f32p(out)),
                    "gm_forward_stack")
        return out

    def run_stack(self, path: int, batch: int, calls: int, layers, first: int = 0):
        """Timed stack passes over device-resident tokens; returns (device ms, wall ms)."""
        arr = (C.c_uint32 * len(layers))(*layers)
        dev, wall = C.c_double(), C.c_double()
        self._check(lib().gm_run_stack(self._h, path, batch, calls, first, arr, len(layers), C.byref(dev),
                                       C.byref(wall)), "gm_run_stack")
        return dev.value, wall.value

    def forward_decode_noalloc(self, layer: int, x_ptr: int, n: int, out_ptr: int, stream: int = 0):
        """Decode-path forward of n <= 8 tokens between device buffers (addresses x_ptr, out_ptr),
        queued on the hipStream_t `stream` (0: the engine's compute stream; 1, hipStreamLegacy: the
        default stream, which torch calls 0); allocates nothing and does not wait."""
        self._check(lib().gm_forward_decode_noalloc(self._h, layer, x_ptr, n, out_ptr, stream or None),
                    "gm_forward_decode_noalloc")

    def read_outputs(self, n: int) -> np.ndarray:
        out = np.empty((n, self.E), np.float32)
        self._check(lib().gm_read_outputs(self._h, _f32p(out), n), "gm_read_outputs")
        return out

    # ---- operators around the layers, on device tensors ------------------------------------------
    # Tensors are torch tensors (or objects with their shape, dtype, stride(), data_ptr() and get_device()) on the
    # engine's GPU; `stream` is a hipStream_t as torch gives it (torch.cuda.current_stream().cuda_stream; 0 is the
    # default stream; None torch's current stream on the engine's GPU, which takes 3 us to look up). Each call queues its
    # work and returns. include/gyro_ops.h states the formulas.

    def _stream(self):
        """Torch's current stream on the engine's GPU, or the default one where torch does not use the GPU."""
        torch = sys.modules.get("torch")
        return torch.cuda.current_stream(self.adapter).cuda_stream if torch and torch.cuda.is_initialized() else 0

    def load_operators(self):
        """Loads the operators' kernels, so that first calls may be captured into a graph."""
        self._check(lib().gm_load_operators(self._h), "gm_load_operators")

    def add_matrix(self, fmt: str, rows: int, cols: int, data, up=None, group: int = 32) -> int:
        """Uploads a 4-bit matrix (or, with `up`, a gated pair) and returns its index. fmt "q4_0" or "q4_1": `data`
        is the uint8 array of its GGUF blocks; "q4": (quants uint8 [rows, cols / 2], scales float16 [rows,
        cols / group], mins float16 or None)."""
        if fmt not in MATRIX_FORMATS:
            raise ValueError(f"matrix format {fmt!r} is none of {sorted(MATRIX_FORMATS)}")
        for value, what in ((rows, "rows"), (cols, "cols"), (group, "group")):
            _count(value, what)
        keep = []

        def parts(m):
            m = m if fmt == "q4" else (m, None, None)
            if len(m) != 3:
                raise ValueError("a q4 matrix is (quants, scales, mins or None)")
            if rows <= 0 or cols <= 0 or group <= 0 or cols % group:
                raise ValueError("a matrix has rows, and columns in whole groups")
            block = {"q4_0": 18, "q4_1": 20}.get(fmt)
            want = [(np.uint8, rows * cols // 32 * block if block else rows * cols // 2),
                    (np.float16, rows * (cols // group)), (np.float16, rows * (cols // group))]
            out = []
            for a, (dtype, size), name in zip(m, want, ("quants", "scales", "mins")):
                if a is not None:
                    a = np.ascontiguousarray(a)
                    if a.dtype != dtype or a.size != size:
                        raise ValueError(f"{name}: {a.dtype} x {a.size}, not {np.dtype(dtype)} x {size}")
                    keep.append(a)
                out.append(None if a is None else a.ctypes.data)
            return out

        d = MatrixDesc(MATRIX_FORMATS[fmt], rows, cols, group, *parts(data), *(parts(up) if up is not None else ()))
        idx = C.c_uint32()
        self._check(lib().gm_add_matrix(self._h, C.byref(d), C.byref(idx)), "gm_add_matrix")
        self._matrices[idx.value] = (rows, cols)
        return idx.value

    def release_matrix(self, matrix: int):
        _count(matrix, "matrix")
        if self._h:
            self._check(lib().gm_release_matrix(self._h, matrix), "gm_release_matrix")
            self._matrices.pop(matrix, None)

    def _rows(self, t, shape, what):
        """(address, stride, type) of a tensor of rows."""
        if t.shape != shape:
            raise ValueError(f"{what}: shape {tuple(t.shape)}, not {shape}")
        if t.get_device() != self.adapter:
            raise ValueError(f"{what}: not on the engine's GPU")
        stride, step = t.stride()
        if step != 1 and shape[1] > 1:
            raise ValueError(f"{what}: the values of a row are not neighbours")
        return t.data_ptr(), stride, _type(t, _ROW_TYPES, what)

    def _flat(self, t, size, types, what):
        """Address of a contiguous tensor of `size` values."""
        if t.numel() != size or not t.is_contiguous():
            raise ValueError(f"{what}: shape {tuple(t.shape)}, not {size} neighbouring values")
        if t.get_device() != self.adapter:
            raise ValueError(f"{what}: not on the engine's GPU")
        _type(t, types, what)
        return t.data_ptr()

    def linear(self, matrix: int, x, y, act: str = "none", accumulate: bool = False, scale: float = 1.0,
               stream: int | None = None):
        """y = act(scale W x) per row (+ y with accumulate), or scale silu(G x) * (U x) of a gated pair."""
        if matrix not in self._matrices:
            raise ValueError(f"no matrix {matrix}")
        rows, cols = self._matrices[matrix]
        n = _count(x.shape[0], "rows of x")
        rc = lib().gm_linear(self._h, matrix, _PACK_ROWS(*self._rows(x, (n, cols), "x"), 0), n,
                             _PACK_ROWS(*self._rows(y, (n, rows), "y"), 0), ACTS[act], accumulate, scale,
                             self._stream() if stream is None else stream)
        if rc:
            self._check(rc, "gm_linear")

    def block_norm(self, h, x, out=None, normed=None, post: bool = False, post_weight=None, post_eps: float = 1e-6,
                   gate=None, gate_act: str = "none", scale: float = 1.0, pre_weight=None, pre_eps: float = 1e-6,
                   stream: int | None = None):
        """out = v = x + scale * gate * a with a = RMSNorm(h) (post) or h, normed = RMSNorm(v). `gate` is [n, 1] (per
        token), [1, E] (per channel) or [n, E]; weights are fp32 [E]. h None: v = x."""
        shape = tuple(x.shape)
        n, E = shape
        _count(n, "rows of x")
        _count(E, "values of a row")
        kind, g = 0, _NO_ROWS
        if gate is not None:
            gs = tuple(gate.shape)
            kind, gs = (GATE_VALUE, shape) if gs == shape else (GATE_CHANNEL, (1, E)) if gs == (1, E) else (GATE_TOKEN, (n, 1))
            g = self._rows(gate, gs, "gate")
        xr = self._rows(x, shape, "x")
        hr = self._rows(h, shape, "h") if h is not None else _NO_ROWS
        out_r = self._rows(out, shape, "out") if out is not None else _NO_ROWS
        nr = self._rows(normed, shape, "normed") if normed is not None else _NO_ROWS
        d = _PACK_NORM(E, post, kind, ACTS[gate_act], *hr, 0, *xr, 0, *out_r, 0, *nr, 0, *g, 0,
                       self._flat(post_weight, E, _FLOAT, "post_weight") if post_weight is not None else 0,
                       self._flat(pre_weight, E, _FLOAT, "pre_weight") if pre_weight is not None else 0,
                       post_eps, pre_eps, scale, 0)
        rc = lib().gm_block_norm(self._h, d, n, self._stream() if stream is None else stream)
        if rc:
            self._check(rc, "gm_block_norm")

    @staticmethod
    def logprobs_workspace(n: int, V: int, top: int = 0) -> int:
        """Bytes of a workspace that suffices for logprobs() of up to n rows of V logits."""
        return lib().gm_logprobs_workspace(_count(n, "n"), _count(V, "V"), _count(top, "top"))

    def logprobs(self, logits, workspace=None, tokens=None, logprob=None, entropy=None, top_ids=None,
                 top_logprobs=None, scale: float = 1.0, stream: int | None = None):
        """Log probabilities of `tokens` (int32 or int64 [n, given]) under softmax(scale * logits) into logprob (fp32
        [n, given]), the entropy (fp32 [n]), and the largest logits' ids (int32 [n, top]) and log probabilities.
        workspace: a uint8 tensor of at least logprobs_workspace() bytes, not shared with calls that may overlap."""
        n, V = logits.shape
        _count(n, "rows of logits")
        _count(V, "logits of a row")
        x = self._rows(logits, (n, V), "logits")
        given = top = wide = ws_bytes = tp = lp = ip = kp = ws = 0
        if tokens is not None:
            if logprob is None:
                raise ValueError("tokens without logprob")
            given = tokens.shape[-1]
            tp = self._flat(tokens, n * given, _INTS, "tokens")
            wide = _type_codes[tokens.dtype] == 4
            lp = self._flat(logprob, n * given, _FLOAT, "logprob")
        elif logprob is not None:
            raise ValueError("logprob without tokens")
        if (top_ids is None) != (top_logprobs is None):
            raise ValueError("top_ids and top_logprobs go together")
        if top_ids is not None:
            top = top_ids.shape[-1]
            ip = self._flat(top_ids, n * top, _INT32, "top_ids")
            kp = self._flat(top_logprobs, n * top, _FLOAT, "top_logprobs")
        if workspace is not None:
            ws_bytes = workspace.numel()
            ws = self._flat(workspace, ws_bytes, _UINT8, "workspace")
        d = _PACK_LOGPROBS(*x, 0, V, given, top, wide, scale, 0, tp, given, lp, given,
                           self._flat(entropy, n, _FLOAT, "entropy") if entropy is not None else 0, ip, kp, top, ws, ws_bytes)
        rc = lib().gm_logprobs(self._h, d, n, self._stream() if stream is None else stream)
        if rc:
            self._check(rc, "gm_logprobs")
