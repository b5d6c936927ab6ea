"""Host mirror of include/m26c_coord.h: the operators between the return of a block and the next token, on device
pointers (for example torch tensor data_ptr()). `Join` holds a block join's plan, `Weights4` a matrix of MXFP4 weights
laid out for the matrix pipe; `token_logprobs` reads a head's logits. A refused call raises CoordError (code 1: bad argument).

The calls launch on `stream` (a hipStream_t as an int, None for the default stream) of the current device and return.
"""
from __future__ import annotations

import ctypes as C

from ._lib import load

ERRLEN = 256


class CoordError(RuntimeError):
    def __init__(self, code: int, what: str):
        super().__init__(f"{what}: error {code}")
        self.code = code


def _ck(code: int, what: str) -> None:
    if code != 0:
        raise CoordError(code, what)


def _int(v: int, what: str) -> int:
    """`v`, refused where C's int would hold another number."""
    if not -0x80000000 <= v <= 0x7FFFFFFF:
        raise CoordError(1, what)
    return v


class _JoinPlan(C.Structure):
    _fields_ = [("cols", C.c_int), ("planes", C.c_int), ("plane_pitch", C.c_long), ("h_pitch", C.c_long), ("norm_pitch", C.c_long),
                ("pre_weight", C.c_void_p), ("post_weight", C.c_void_p), ("gate_cols", C.c_int), ("gate_pitch", C.c_long),
                ("scale", C.c_float), ("eps", C.c_float), ("payload_pitch", C.c_size_t), ("scales_pitch", C.c_size_t)]


class Join:
    """h' = h + scale * gate * norm(sum of planes); n = norm(h'). Pitches default to contiguous rows; `gate_cols` is 0 (no
    gate), 1 (a value per row) or `cols`, and `gate_pitch` 0 repeats one gate for all rows. `post_weight` None leaves
    the norm after the block out."""

    def __init__(self, cols: int, pre_weight: int | None, post_weight: int | None = None, planes: int = 1, gate_cols: int = 0,
                 gate_pitch: int = 0, scale: float = 1.0, eps: float = 1e-6, plane_pitch: int = 0, h_pitch: int = 0,
                 norm_pitch: int = 0, payload_pitch: int = 0, scales_pitch: int = 0):
        for v in (cols, planes, gate_cols):
            _int(v, "block join")
        self._plan = _JoinPlan(cols, planes, plane_pitch or cols, h_pitch or cols, norm_pitch or cols, pre_weight, post_weight, gate_cols,
                               gate_pitch, scale, eps, payload_pitch or cols, scales_pitch or cols // 32)
        self._ref = C.byref(self._plan)
        self._planes, self._rest = planes, (None,) * (4 - planes)
        self._call = load().m26c_block_join

    def __call__(self, rows: int, h: int, planes, h_out: int | None, norm: int | None = None, gate: int | None = None,
                 payload: int | None = None, scales: int | None = None, stream: int | None = None) -> None:
        """`planes`: that many BF16 pointers. `h_out` may be `h`. Any of `h_out`, `norm` and `payload` with `scales` may
        be None, as long as one is not."""
        if len(planes) != self._planes:
            raise CoordError(1, f"block join of {self._planes} planes called with {len(planes)}")
        rc = self._call(self._ref, rows, h, *planes, *self._rest, gate, h_out, norm, payload, scales, stream)
        if rc:
            raise CoordError(rc, "block join")


class Weights4:
    """[n][k] MXFP4 weights (payload [n][k / 2], low nibble = even k, 16-byte aligned; one E8M0 byte per 32 k, at any alignment), laid
    out once on the current device; the sources may be freed afterwards."""

    def __init__(self, payload: int, scales: int, n: int, k: int, stream: int | None = None):
        self._h = C.c_void_p()
        self.n, self.k = n, k
        buf = C.create_string_buffer(ERRLEN)
        rc = load().m26c_w4_new(payload, scales, n, k, stream, C.byref(self._h), buf, ERRLEN)
        if rc:
            raise CoordError(rc, buf.value.decode("utf-8", "replace"))
        self._bf16, self._fp8 = load().m26c_w4_matvec, load().m26c_w4_matvec_fp8

    def matvec(self, x: int, rows: int, y: int, y_bf16: bool = False, x_pitch: int = 0, y_pitch: int = 0, stream: int | None = None) -> None:
        """y = x W^T for `rows` BF16 rows; FP32 out, or BF16."""
        _ck(self._bf16(self._h, x, x_pitch or self.k, _int(rows, "w4 product"), y, y_bf16, y_pitch or self.n, stream), "w4 product")

    def matvec_fp8(self, payload: int, scales: int, rows: int, y: int, y_bf16: bool = False, payload_pitch: int = 0,
                   scales_pitch: int = 0, y_pitch: int = 0, stream: int | None = None) -> None:
        """The same for wire rows (E4M3 codes, one UE8M0 byte per 32 values)."""
        _ck(self._fp8(self._h, payload, payload_pitch or self.k, scales, scales_pitch or self.k // 32, _int(rows, "w4 product of wire rows"), y,
                      y_bf16, y_pitch or self.n, stream), "w4 product of wire rows")

    def close(self) -> None:
        if getattr(self, "_h", None) and self._h.value and load is not None:  # load is gone at interpreter exit
            load().m26c_w4_free(self._h)
            self._h = C.c_void_p()

    __del__ = close


def token_logprobs_workspace(rows: int, vocab: int, top: int) -> int:
    """Bytes of device memory token_logprobs needs for these sizes (0: none)."""
    if max(rows, vocab, top) > 0x7FFFFFFF or min(rows, vocab, top) < 0:
        return 0
    return int(load().m26c_token_logprobs_workspace(rows, vocab, top))


def token_logprobs(logits: int, bf16: bool, rows: int, vocab: int, pitch: int, given: int | None, n_given: int, given_logprob: int | None,
                   entropy: int | None, top: int, top_ids: int | None, top_logprob: int | None, workspace: int | None,
                   workspace_bytes: int, scale: float = 1.0, stream: int | None = None) -> None:
    """Log softmax of scale * logits at `given` [rows][n_given] (int32; an id outside the vocabulary gives NaN), its entropy per
    row and its `top` largest values with their ids (-1 where masked logits leave fewer)."""
    for v in (rows, vocab, n_given, top):
        _int(v, "token log probabilities")
    _ck(load().m26c_token_logprobs(logits, bf16, pitch, rows, vocab, scale, given, n_given, given_logprob, entropy, top, top_ids,
                                   top_logprob, workspace, workspace_bytes, stream), "token log probabilities")
