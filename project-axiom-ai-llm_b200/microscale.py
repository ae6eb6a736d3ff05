"""Microscaled operands from Python: expert weights and activations in 4 bits, activation
checkpoints in 8 bits (formats in include/axm_moe.h).

    quantize_rows(x) -> Mx4Rows             dequantize_rows(q) -> x
    quantize_weights(w) -> Mx4Weights       dequantize_weights(q) -> w
    quantize_rows8(x) -> (codes, scales)    dequantize_rows8(codes, scales) -> x
    Mx4Linear        y = q4(x) . W^T for one weight matrix
    Mx4ExpertFfn     the expert feed-forward over a segment table
    Mx4MoeLayer      the whole layer (MoeLayer's call) with expert weights in 4 bits
    Mx8TrainFfn      the expert feed-forward's training step, g and u kept in 8 bits between its passes

Like the rest of the package these are thin callers of the C ABI: tensors are device memory,
work goes to the current stream, nothing synchronises.  The engine keeps its weights in bf16
with fp32 masters (core/src/CUDA/util/gpu_types.cuh:148-168); either is a source here.
"""
import ctypes
import functools
import importlib
import inspect

import torch

_pkg = importlib.import_module(__package__)

_DTYPES = {torch.bfloat16: _pkg.DTYPE_BF16, torch.float32: _pkg.DTYPE_FP32}


def _dtype(t):
    if t not in _DTYPES:
        raise TypeError(f"bf16 or fp32 is needed, not {t}")
    return _DTYPES[t]


def _on_its_device(call):
    """The library enqueues on the current device: makes that the device of the call's first tensor (or of
    the object's)."""
    name = next(iter(inspect.signature(call).parameters))

    @functools.wraps(call)
    def wrapped(*args, **kw):
        first = args[0] if args else kw.get(name)
        index = None if first is None else first.device.index
        if index is None or index == torch.cuda.current_device():  # host tensors are refused inside
            return call(*args, **kw)
        with torch.cuda.device(first.device):
            return call(*args, **kw)
    return wrapped


def _rows_of(x):
    if not x.is_cuda or x.dim() != 2:
        raise ValueError("a CUDA matrix with contiguous rows is needed")
    rows, k = x.shape
    ld, one = x.stride()
    if one != 1 and k > 1:
        raise ValueError("a CUDA matrix with contiguous rows is needed")
    return rows, k, ld if rows > 1 else k  # one row has no next one: its stride says nothing


def _check_index(t, width, device, what):
    """An int32 device tensor as the kernels read it: [n], or [n][width].  (None: not given.)"""
    if t is None:
        return
    if t.dtype != torch.int32 or t.device != device or not t.is_contiguous() or \
            (t.dim() != 1 if width is None else t.dim() != 2 or t.shape[1] != width):
        raise ValueError(f"{what}: a contiguous int32 {'[n]' if width is None else f'[n][{width}]'} on {device} is needed, "
                         f"not {t.dtype} {tuple(t.shape)} on {t.device}")


def _check_out(out, shape, device, dtype=None):
    if tuple(out.shape) != tuple(shape) or not out.is_contiguous() or out.device != device or \
            (dtype is not None and out.dtype != dtype):
        raise ValueError(f"out: a contiguous {'' if dtype is None else dtype} {tuple(shape)} on {device} is needed, "
                         f"not {out.dtype} {tuple(out.shape)} on {out.device}")


def _address(t):
    return None if t is None else t.data_ptr()


def _bytes(call, *args):
    a, b = ctypes.c_size_t(0), ctypes.c_size_t(0)
    _pkg.check(call(*args, ctypes.byref(a), ctypes.byref(b)))
    return a.value, b.value


class Mx4Rows:
    """Rows in 4 bits: codes [rows][K/2], tile-ordered scales, the segment table they follow.  Both
    lie in one buffer, the scales from `scales_at` on."""

    def __init__(self, buffer, scales_at, rows, k, segments=None):
        self.buffer, self.scales_at, self.rows, self.k, self.segments = buffer, scales_at, rows, k, segments

    @property
    def codes(self):
        return self.buffer[:self.rows * (self.k // 2)].view(self.rows, self.k // 2)

    @property
    def scales(self):
        return self.buffer[self.scales_at:]

    @property
    def device(self):
        return self.buffer.device


class Mx4Weights:
    """Weights in 4 bits: codes [E][N][K/2], tile-ordered scales."""

    def __init__(self, codes, scales, experts, k, n):
        self.codes, self.scales, self.experts, self.k, self.n = codes, scales, experts, k, n
        self.device = codes.device

    @classmethod
    def from_checkpoint(cls, codes, scales):
        """From codes [E][N][K/2] and scale bytes [E][N][K/32], as 4-bit checkpoints keep them.
        The codes are used as they are, the scale bytes are brought into the tiles' order."""
        lib = _pkg.load()
        if not (codes.is_cuda and scales.is_cuda and codes.device == scales.device and
                codes.is_contiguous() and scales.is_contiguous() and
                codes.dtype == torch.uint8 and scales.dtype == torch.uint8 and codes.dim() == 3):
            raise ValueError("contiguous uint8 CUDA tensors [E][N][K/2] and [E][N][K/32] on one device are needed")
        e, n, k = codes.shape[0], codes.shape[1], 2 * codes.shape[2]
        if scales.shape != (e, n, k // 32):
            raise ValueError(f"scales {tuple(scales.shape)} do not belong to codes {tuple(codes.shape)}")
        _, size = _bytes(lib.axm_mx4_weights_bytes, e, k, n)
        with torch.cuda.device(codes.device):
            packed = torch.empty(size, dtype=torch.uint8, device=codes.device)
            _pkg.check(lib.axm_mx4_pack_scales(scales.data_ptr(), e, k, n, packed.data_ptr(),
                                               _pkg.raw_stream(codes.device.index)))
        return cls(codes, packed, e, k, n)


@_on_its_device
def quantize_rows(x, segments=None, row_src=None, row_div=1):
    """x [rows][K] bf16 or fp32 to 4 bits; row_src: row r is read from x[row_src[r] // row_div], which has to
    exist (negative: zeros).  Rows that no segment covers cannot be read back."""
    rows, k, ld = _rows_of(x)
    nseg = 0
    if row_src is not None:
        _check_index(row_src, None, x.device, "row_src")
        rows = row_src.numel()
    if segments is not None:
        _check_index(segments, 4, x.device, "segments")
        nseg = segments.shape[0]
        if nseg == 0:  # an empty tensor has no address, which would mean that all rows form one segment
            raise ValueError("segments: an empty table")
    # the sizes of axm_mx4_rows_bytes; sizes that it refuses are refused by the call below
    at = (rows * (k // 2) + 255) & -256
    size = at + (rows // 128 + (nseg or 1)) * ((k + 255) >> 8) * 1024
    device = x.device
    buffer = torch.empty(size, dtype=torch.uint8, device=device)
    base = buffer.data_ptr()
    status = _pkg.load().axm_mx4_quantize_rows(x.data_ptr(), _dtype(x.dtype), ld, _address(row_src), row_div, rows, k,
                                               _address(segments), nseg, base, base + at, _pkg.raw_stream(device.index))
    if status:
        _pkg.check(status)
    return Mx4Rows(buffer, at, rows, k, segments)


@_on_its_device
def dequantize_rows(q, dtype=torch.bfloat16, out=None):
    """Rows that no segment covers are not written: without `out` they hold what the allocator gave."""
    buffer, rows, k, ld = q.buffer, q.rows, q.k, q.k
    device = buffer.device
    if out is None:
        out = torch.empty((rows, k), dtype=dtype, device=device)
    else:
        got = _rows_of(out)
        if got[:2] != (rows, k) or out.device != device:
            raise ValueError(f"out is {tuple(out.shape)} on {out.device}, the rows are {(rows, k)} on {device}")
        dtype, ld = out.dtype, got[2]
    segments = q.segments
    base = buffer.data_ptr()
    status = _pkg.load().axm_mx4_dequantize_rows(base, base + q.scales_at, rows, k, _address(segments),
                                                 0 if segments is None else segments.shape[0], out.data_ptr(),
                                                 _dtype(dtype), ld, _pkg.raw_stream(device.index))
    if status:
        _pkg.check(status)
    return out


@_on_its_device
def quantize_rows8(x):
    """x [rows][K] to 8 bits: codes [rows][K] (e4m3), scale bytes [rows][K/32]."""
    rows, k, ld = _rows_of(x)
    device = x.device
    codes = torch.empty((rows, k), dtype=torch.uint8, device=device)
    scales = torch.empty((rows, k // 32), dtype=torch.uint8, device=device)
    _pkg.check(_pkg.load().axm_mx8_quantize_rows(x.data_ptr(), _dtype(x.dtype), ld, rows, k, codes.data_ptr(),
                                                 scales.data_ptr(), _pkg.raw_stream(device.index)))
    return codes, scales


@_on_its_device
def dequantize_rows8(codes, scales, dtype=torch.bfloat16):
    rows, k = codes.shape
    device = codes.device
    if not (codes.is_cuda and codes.is_contiguous() and scales.is_contiguous() and scales.shape == (rows, k // 32) and
            scales.device == device and codes.dtype == scales.dtype == torch.uint8):
        raise ValueError("contiguous uint8 codes [rows][K] and scales [rows][K/32] on one CUDA device are needed")
    out = torch.empty((rows, k), dtype=dtype, device=device)
    _pkg.check(_pkg.load().axm_mx8_dequantize_rows(codes.data_ptr(), scales.data_ptr(), rows, k, out.data_ptr(),
                                                   _dtype(dtype), k, _pkg.raw_stream(device.index)))
    return out


@_on_its_device
def quantize_weights(w):
    """w [E][K][N] bf16 or fp32 (the engine's layout, K is summed over) to 4 bits."""
    if not (w.is_cuda and w.dim() == 3 and w.is_contiguous()):
        raise ValueError("a contiguous CUDA tensor [E][K][N] is needed")
    e, k, n = w.shape
    device = w.device
    codes = torch.empty((e, n, k // 2), dtype=torch.uint8, device=device)
    # the size of axm_mx4_weights_bytes; sizes that it refuses are refused by the call below
    scales = torch.empty(e * ((n + 127) >> 7) * ((k + 255) >> 8) * 1024, dtype=torch.uint8, device=device)
    _pkg.check(_pkg.load().axm_mx4_quantize_weights(w.data_ptr(), _dtype(w.dtype), e, k, n, codes.data_ptr(),
                                                    scales.data_ptr(), _pkg.raw_stream(device.index)))
    return Mx4Weights(codes, scales, e, k, n)


@_on_its_device
def dequantize_weights(q, dtype=torch.bfloat16):
    device = q.device
    w = torch.empty((q.experts, q.k, q.n), dtype=dtype, device=device)
    _pkg.check(_pkg.load().axm_mx4_dequantize_weights(q.codes.data_ptr(), q.scales.data_ptr(), q.experts, q.k, q.n,
                                                      w.data_ptr(), _dtype(dtype), _pkg.raw_stream(device.index)))
    return w


class _Workspace:
    """Scratch of one object; its first word is the status word."""

    def _scratch(self, size, device):
        self.device = device
        self.workspace = torch.empty(max(size, 256), dtype=torch.uint8, device=device)
        self.workspace[:4].zero_()  # the status word, until the first call

    def status(self):
        """Reads the status word of the last call (synchronises): 0, or the code of a kernel whose
        bounded wait gave up."""
        torch.cuda.synchronize(self.workspace.device)
        return int(self.workspace[:4].view(torch.int32).item())


class Mx4Linear(_Workspace):
    """y = q4(x) . W^T with W ([1][N][K/2] in 4 bits) and scratch for up to `tokens` rows."""

    def __init__(self, weights, tokens):
        if weights.experts != 1:
            raise ValueError("one weight matrix is needed")
        self.lib, self.w, self.tokens = _pkg.load(), weights, tokens
        n = ctypes.c_size_t(0)
        _pkg.check(self.lib.axm_mx4_linear_workspace_bytes(tokens, weights.k, weights.n, ctypes.byref(n)))
        self._scratch(n.value, weights.codes.device)

    @_on_its_device
    def forward(self, x, out=None, dtype=torch.bfloat16):
        w, device = self.w, self.device
        rows, k, ld = _rows_of(x)
        if rows > self.tokens or k != w.k or x.device != device:
            raise ValueError(f"x {tuple(x.shape)} on {x.device}: up to {self.tokens} rows of {w.k} on {device}")
        if out is None:
            out = torch.empty((rows, w.n), dtype=dtype, device=device)
        else:
            _check_out(out, (rows, w.n), device)
        status = self.lib.axm_mx4_linear(x.data_ptr(), _dtype(x.dtype), ld, rows, k, w.n, w.codes.data_ptr(),
                                         w.scales.data_ptr(), out.data_ptr(), _dtype(out.dtype),
                                         self.workspace.data_ptr(), self.workspace.numel(),
                                         _pkg.raw_stream(device.index))
        if status:
            _pkg.check(status)
        return out


def _expert_table(gate, up, down):
    if (gate.experts, gate.k, gate.n) != (up.experts, up.k, up.n) or \
            (down.experts, down.k, down.n) != (gate.experts, gate.n, gate.k):
        raise ValueError("gate and up are [E][F][D/2], down is [E][D][F/2]")
    for w in (up, down):
        if w.device != gate.device:
            raise ValueError(f"weights on {gate.device} and {w.device}: one device is needed")
    return _pkg.Mx4ExpertWeights(*(t.data_ptr() for w in (gate, up, down) for t in (w.codes, w.scales)))


class Mx4ExpertFfn(_Workspace):
    """The expert feed-forward from 4-bit weights over up to `rows` rows in up to `segments`
    segments (default: one per expert); `tokens`, the most rows a segment is expected to have, guides the
    choice of kernel."""

    def __init__(self, gate, up, down, rows, tokens, segments=None):
        self.lib = _pkg.load()
        self.weights = (gate, up, down)
        self.table = _expert_table(gate, up, down)
        self.rows, self.segments = rows, gate.experts if segments is None else segments
        self.desc = _pkg.make_desc(tokens, gate.k, gate.n, gate.experts, 1, flags=0)
        n = ctypes.c_size_t(0)
        _pkg.check(self.lib.axm_mx4_expert_ffn_workspace_bytes(ctypes.byref(self.desc), rows, self.segments,
                                                               ctypes.byref(n)))
        self._scratch(n.value, gate.codes.device)

    @_on_its_device
    def forward(self, x, segments, out=None, dtype=torch.bfloat16):
        """x [rows][D] bf16, segments int32 [n][4] {a_row0, out_row0, rows, expert} (device).  Rows that no
        segment covers are not written: without `out` they hold what the allocator gave."""
        rows, d, _ = _rows_of(x)
        dev = self.device
        if rows > self.rows or d != self.desc.d_model or not x.is_contiguous() or x.dtype != torch.bfloat16 or x.device != dev:
            raise ValueError(f"x: up to {self.rows} contiguous bf16 rows of {self.desc.d_model} on {dev}")
        _check_index(segments, 4, dev, "segments")
        if segments.shape[0] > self.segments:
            raise ValueError(f"segments: {segments.shape[0]}, up to {self.segments} were announced")
        if out is None:
            out = torch.empty(rows, d, dtype=dtype, device=dev)
        else:
            _check_out(out, x.shape, dev)
        _pkg.check(self.lib.axm_mx4_expert_ffn(ctypes.byref(self.desc), x.data_ptr(), rows, segments.data_ptr(),
                                               segments.shape[0], ctypes.byref(self.table), out.data_ptr(),
                                               _dtype(out.dtype), self.workspace.data_ptr(), self.workspace.numel(),
                                               _pkg.raw_stream(dev.index)))
        return out


class Mx4MoeLayer(_Workspace):
    """MoeLayer with expert weights in 4 bits.  weights: router_w (and router_bias) as for MoeLayer;
    gate, up, down (and shared_gate, shared_up, shared_down) Mx4Weights."""

    def __init__(self, weights, tokens, top_k, residual=True, hist_accumulate=False):
        self.lib, self.w = _pkg.load(), weights
        wr, gate = weights["router_w"], weights["gate"]
        self.experts = _expert_table(gate, weights["up"], weights["down"])
        self.shared = None
        shared = 0
        if weights.get("shared_gate") is not None:
            self.shared = _expert_table(weights["shared_gate"], weights["shared_up"], weights["shared_down"])
            shared = weights["shared_gate"].experts
            if (weights["shared_gate"].k, weights["shared_gate"].n) != (gate.k, gate.n):
                raise ValueError("shared experts have the routed experts' sizes")
        bias = weights.get("router_bias")
        for t in [wr, gate, weights.get("shared_gate"), bias]:
            if t is not None and t.device != gate.device:
                raise ValueError(f"weights on {gate.device} and {t.device}: one device is needed")
        if not wr.is_contiguous() or wr.dtype not in _DTYPES:
            raise ValueError("router_w: a contiguous bf16 or fp32 matrix is needed")
        if bias is not None and (bias.numel() != gate.experts or not bias.is_contiguous() or bias.dtype != torch.float32):
            raise ValueError(f"router_bias: {gate.experts} contiguous fp32 values are needed")
        if wr.shape != (gate.k, gate.experts):
            raise ValueError(f"router_w {tuple(wr.shape)}: [D][E] = {(gate.k, gate.experts)} is needed")
        flags = (_pkg.FLAG_RESIDUAL if residual else 0) | (_pkg.FLAG_HIST_ACCUMULATE if hist_accumulate else 0)
        self.desc = _pkg.make_desc(tokens, gate.k, gate.n, gate.experts, top_k, shared,
                                   _pkg.ROUTER_FP32 if wr.dtype == torch.float32 else _pkg.ROUTER_BF16, flags)
        n = ctypes.c_size_t(0)
        _pkg.check(self.lib.axm_moe_mx4_workspace_bytes(ctypes.byref(self.desc), ctypes.byref(n)))
        dev = wr.device
        self._scratch(n.value, dev)
        self.T, self.D, self.k = tokens, gate.k, top_k
        self.topk_idx = torch.empty(tokens, top_k, dtype=torch.int32, device=dev)
        self.topk_gate = torch.empty(tokens, top_k, dtype=torch.float32, device=dev)
        self.histogram = torch.zeros(gate.experts, dtype=torch.int32, device=dev)

    @_on_its_device
    def forward(self, x, out=None):
        """out = x + sum of the chosen experts' outputs (without residual: the sum), histogram."""
        dev = self.device
        if x.shape != (self.T, self.D) or x.dtype != torch.bfloat16 or not x.is_contiguous() or x.device != dev:
            raise ValueError(f"x: contiguous bf16 {(self.T, self.D)} on {dev}")
        if out is None:
            out = torch.empty_like(x)
        else:
            _check_out(out, x.shape, dev, torch.bfloat16)
        t = _pkg.MoeTensors()
        t.x, t.out, t.router_w = x.data_ptr(), out.data_ptr(), self.w["router_w"].data_ptr()
        if self.w.get("router_bias") is not None:
            t.router_bias = self.w["router_bias"].data_ptr()
        t.topk_idx, t.topk_gate = self.topk_idx.data_ptr(), self.topk_gate.data_ptr()
        t.histogram = self.histogram.data_ptr()
        _pkg.check(self.lib.axm_moe_forward_mx4(ctypes.byref(self.desc), ctypes.byref(t), ctypes.byref(self.experts),
                                                None if self.shared is None else ctypes.byref(self.shared),
                                                self.workspace.data_ptr(), self.workspace.numel(),
                                                _pkg.raw_stream(dev.index)))
        return out, self.histogram


class Mx8TrainFfn:
    """Training step of the expert feed-forward: forward(x, segments) -> o keeps the gate's and the up
    projection's outputs in 8 bits, backward(d_o) gives the gradients from them.

    gate, up [E][D][F] and down [E][F][D] bf16; up to `rows` rows, segments padded to 64 rows with zero
    rows (the layer's training layout).  dtype: of o and of every gradient.  Rows that no segment covers are
    not written: d_x, and o without `out`, hold there what the allocator gave (the gradients of experts that
    a table leaves out are zero).  What is kept is in `checkpoint`; `scratch` (h, dG, dU) holds nothing
    between calls and may be shared by objects of the same sizes that run one after the other on one stream."""

    def __init__(self, gate, up, down, rows, dtype=torch.bfloat16, scratch=None):
        self.lib = _pkg.load()
        e, d, f = gate.shape
        if up.shape != (e, d, f) or down.shape != (e, f, d):
            raise ValueError("gate and up are [E][D][F], down is [E][F][D]")
        for w in (gate, up, down):
            if w.dtype != torch.bfloat16 or not w.is_contiguous() or not w.is_cuda or w.device != gate.device:
                raise ValueError("contiguous bf16 CUDA weights on one device are needed")
        dev = self.device = gate.device
        self.weights, self.rows, self.dtype = (gate, up, down), rows, dtype
        _dtype(dtype)
        self.desc = _pkg.make_desc(rows, d, f, e, 1, flags=0)
        _bytes(self.lib.axm_mx8_checkpoint_bytes, rows, f)  # refuses sizes that cannot be kept
        self.checkpoint = [torch.empty(rows, n, dtype=torch.uint8, device=dev) for n in (f, f // 32, f, f // 32)]
        self.keep = _pkg.Mx8Checkpoint(*(t.data_ptr() for t in self.checkpoint))
        if scratch is not None:
            if len(scratch) != 3:
                raise ValueError("scratch: three matrices are needed")
            for t in scratch:
                _check_out(t, (rows, f), dev, torch.bfloat16)
        self.scratch = scratch or [torch.empty(rows, f, dtype=torch.bfloat16, device=dev) for _ in range(3)]
        self.status_word = torch.zeros(1, dtype=torch.int32, device=dev)
        self.saved = None

    def status(self):
        """Reads the status word (synchronises); sticky until it is cleared by the caller."""
        torch.cuda.synchronize(self.status_word.device)
        return int(self.status_word.item())

    def _check(self, t, what):
        if t.shape[0] > self.rows or t.shape[1] != self.desc.d_model or t.dtype != torch.bfloat16 or \
                not t.is_contiguous() or t.device != self.status_word.device:
            raise ValueError(f"{what}: up to {self.rows} contiguous bf16 rows of {self.desc.d_model} on {self.status_word.device}")

    @_on_its_device
    def forward(self, x, segments, out=None):
        self._check(x, "x")
        _check_index(segments, 4, x.device, "segments")
        if out is None:
            out = torch.empty(x.shape, dtype=self.dtype, device=x.device)
        else:
            _check_out(out, x.shape, x.device)
        p = _address
        _pkg.check(self.lib.axm_mx8_expert_ffn_train(
            ctypes.byref(self.desc), p(x), x.shape[0], p(segments), segments.shape[0], *map(p, self.weights),
            ctypes.byref(self.keep), p(self.scratch[0]), p(out), _dtype(out.dtype), p(self.status_word),
            _pkg.raw_stream(self.device.index)))
        self.saved = (x, segments)
        return out

    @_on_its_device
    def backward(self, d_o, weight_grads=True):
        """{d_x, d_gate, d_up, d_down} (weight_grads False: d_x alone) of the last forward call."""
        if self.saved is None:
            raise RuntimeError("backward before forward")
        x, segments = self.saved
        self._check(d_o, "d_o")
        if d_o.shape != x.shape:
            raise ValueError(f"d_o {tuple(d_o.shape)} is not like x {tuple(x.shape)}")
        p = _address
        grads = {"d_x": torch.empty(x.shape, dtype=self.dtype, device=x.device)}
        if weight_grads:  # experts that the table leaves out are not written: zero
            make = torch.empty if segments.shape[0] >= self.desc.num_experts else torch.zeros
            for n, w in zip(("d_gate", "d_up", "d_down"), self.weights):
                grads[n] = make(w.shape, dtype=self.dtype, device=x.device)
        _pkg.check(self.lib.axm_mx8_expert_ffn_backward(
            ctypes.byref(self.desc), p(x), x.shape[0], p(segments), segments.shape[0], ctypes.byref(self.keep), p(d_o),
            *map(p, self.weights), *map(p, self.scratch), p(grads["d_x"]), p(grads.get("d_gate")),
            p(grads.get("d_up")), p(grads.get("d_down")), _dtype(self.dtype), p(self.status_word),
            _pkg.raw_stream(self.device.index)))
        return grads
