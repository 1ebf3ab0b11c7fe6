"""Operators over sequences, in the manner of the Device* classes: the gated
linear recurrence with its backward pass and single-token step
(DeviceLinearRecurrence), and beam search's selection and reordering of states
(DeviceBeamSearch).

The reference has no counterpart.  Buffers are CUDA torch tensors of float32,
float16 or bfloat16 (states and scores float32); calls are recorded into a
CommandList and run when it is committed to a Stream.  A recorded call keeps
its tensors alive until it has run; as everywhere in this package, a program
that uses several streams orders them itself.
"""
from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib as L
from .primitives import _Module, _nbytes, synchronize

_FLOATS = {torch.float32: L.F32, torch.float16: L.F16, torch.bfloat16: L.BF16}
_GATES = {"linear": L.GATE_LINEAR, "sigmoid": L.GATE_SIGMOID}
_F32, _I32, _INT32, _U8 = (torch.float32,), (torch.int32,), (torch.int32, torch.uint32), (torch.uint8, torch.bool)

# A call for one token takes the GPU a few microseconds, so the checks below are written to take the host no
# longer than that: one read of each property, no containers built for what is in order.


def _float_dtype(first: torch.Tensor, *others: Optional[torch.Tensor]) -> int:
    """lcpp_dtype of tensors that all have the same floating element type."""
    dtype = first.dtype
    for t in others:
        if t is not None and t.dtype != dtype:
            raise TypeError(f"matrices must have the same element type, not {dtype} and {t.dtype}")
    try:
        return _FLOATS[dtype]
    except KeyError:
        raise TypeError(f"unsupported element type {dtype}") from None


def _gate(mode) -> int:
    try:
        return _GATES[mode]
    except KeyError:
        raise ValueError(f"mode must be 'linear' or 'sigmoid', not {mode!r}") from None


def _one_device(*tensors: Optional[torch.Tensor]) -> None:
    device = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != device:
            raise ValueError("all buffers of a call must be on one device")
    if device < 0:
        raise ValueError("buffers must be CUDA tensors")


def _matrix(t: torch.Tensor, name: str):
    """(pointer, row stride, rows, channels) of a (rows, channels) or (batch, time, channels) tensor whose
    rows are one stride apart and whose channels are adjacent."""
    shape = t.shape
    if len(shape) == 2:
        rows, channels = shape
        row, unit = t.stride()
    elif len(shape) == 3:
        batch, time, channels = shape
        outer, row, unit = t.stride()
        rows = batch * time
        if time == 1:
            row = outer
        elif batch > 1 and rows and outer != time * row:
            raise ValueError(f"{name}: the batch stride must be the row stride times the length")
    else:
        raise ValueError(f"{name} must have the shape (rows, channels) or (batch, time, channels)")
    if unit != 1 and channels > 1 and rows:
        raise ValueError(f"{name}: the channels of a row must be adjacent")
    if row < channels and rows > 1:
        raise ValueError(f"{name}: rows must not overlap")
    return t.data_ptr(), row, rows, channels


def _like(t: Optional[torch.Tensor], first: torch.Tensor, rows: int, channels: int, name: str):
    """(pointer, row stride) of a matrix of the first one's size (None: a null pointer)."""
    if t is None:
        return None, 0
    if t.shape == first.shape and t.is_contiguous():  # the usual one
        return t.data_ptr(), channels
    pointer, row, r, c = _matrix(t, name)
    if r != rows or c != channels:
        raise ValueError(f"{name} must have the same shape as the call's other matrices, "
                         f"{(rows, channels)}, not {(r, c)}")
    return pointer, row


def _dense(t: Optional[torch.Tensor], shape, dtypes, name: str) -> Optional[int]:
    """Pointer of a contiguous tensor of this shape and one of these types (None stays None)."""
    if t is None:
        return None
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must have the element type {dtypes[0]}")
    if t.shape != shape:
        raise ValueError(f"{name} must have the shape {tuple(shape)}, not {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def _temp(t: Optional[torch.Tensor]):
    """(pointer, bytes) of the temp buffer."""
    if t is None:
        return None, 0
    if not t.is_contiguous():
        raise ValueError("temp_storage must be contiguous")
    return t.data_ptr(), _nbytes(t)


class _Recorded(_Module):
    def _call(self, cmdlist, entry, args, keep, what) -> None:
        """Record entry(*args, stream); `keep`: the tensors that it uses."""

        def run(stream, keep=keep):
            status = entry(*args, stream)
            if status:
                raise L.LcppError(status, what)

        cmdlist.append(run)
        if self._debug_stream is not None:  # debug: commit + synchronize at once
            self._debug_stream << cmdlist.commit() << synchronize()


class DeviceLinearRecurrence(_Recorded):
    """h_t = a_t h_{t-1} + b_t per channel, along the rows of each sequence.

    mode "linear":  d_gate = a, d_in = b; the product of the gates along up to 128 rows must stay finite
    mode "sigmoid": a = sigmoid(d_gate), b = (1 - a) d_in

    Matrices are (rows, channels) or (batch, time, channels), channels adjacent, any row stride.
    offsets_or_length: the length of every sequence (rows must be a multiple of it), or S + 1 ascending int32 /
    uint32 row offsets on the device (CSR) of S sequences; rows outside them are padding (zeros come out).
    States are float32 of the shape (S, channels).  temp_storage is contiguous and 16-byte aligned, as temp_buffer's is.
    """

    @staticmethod
    def GetTempStorageBytes(num_rows: int, num_channels: int) -> int:
        return int(L.lib().lcpp_linear_recurrence_temp_bytes(num_rows, num_channels))

    @staticmethod
    def GetSavedStateBytes(num_rows: int, num_channels: int) -> int:
        """Bytes of d_saved, which Forward fills for Backward."""
        return int(L.lib().lcpp_linear_recurrence_saved_bytes(num_rows, num_channels))

    @staticmethod
    def _sequences(sequences: Union[int, torch.Tensor], rows: int):
        """(count, length, offsets pointer)."""
        if isinstance(sequences, torch.Tensor):
            if sequences.dtype not in _INT32:
                raise TypeError("offsets must hold 32-bit integers")
            if sequences.dim() != 1 or sequences.numel() < 1 or not sequences.is_contiguous():
                raise ValueError("offsets must be a contiguous vector of num_sequences + 1 row offsets")
            return sequences.numel() - 1, 0, sequences.data_ptr()
        length = int(sequences)
        if length < 0 or (rows % length if length else rows):
            raise ValueError(f"{rows} rows are no whole number of sequences of length {length}")
        return (rows // length if length else 0), length, None

    @staticmethod
    def _init(d_init, count: int, channels: int):
        """(pointer, stride) of the initial states; an expanded (stride 0) state serves all sequences."""
        if d_init is None:
            return None, 0
        if d_init.dtype != torch.float32:
            raise TypeError("d_init must have the element type torch.float32")
        if d_init.shape != (count, channels):
            raise ValueError(f"d_init must have the shape {(count, channels)}, not {tuple(d_init.shape)}")
        if channels > 1 and count and d_init.stride(1) != 1:
            raise ValueError("d_init: the channels of a state must be adjacent")
        return d_init.data_ptr(), d_init.stride(0)

    def Forward(self, cmdlist, temp_storage, d_gate, d_in, d_out, offsets_or_length, d_init=None, d_last=None,
                d_saved=None, mode="sigmoid"):
        """d_out = h; d_last = h after each sequence's last row (d_init for an empty sequence).  d_out may be
        d_gate or d_in (with the same row stride), and d_last may be d_init; other overlaps are refused."""
        dt, gate = _float_dtype(d_gate, d_in, d_out), _gate(mode)
        offsets = offsets_or_length if isinstance(offsets_or_length, torch.Tensor) else None
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_gate, d_in, d_out, d_init, d_last, d_saved, temp_storage, offsets)
        _one_device(*keep)
        pg, sg, rows, channels = _matrix(d_gate, "d_gate")
        pi, si = _like(d_in, d_gate, rows, channels, "d_in")
        po, so = _like(d_out, d_gate, rows, channels, "d_out")
        count, length, off = self._sequences(offsets_or_length, rows)
        p0, s0 = self._init(d_init, count, channels)
        pl = _dense(d_last, (count, channels), _F32, "d_last")
        ps = _saved(d_saved, rows, channels)
        self._call(cmdlist, L.lib().lcpp_linear_recurrence_forward,
                   (gate, dt, pg, sg, pi, si, po, so, rows, channels, count, length, off, p0, s0, pl, ps,
                    temp, temp_bytes),
                   keep, "DeviceLinearRecurrence.Forward")

    def Backward(self, cmdlist, temp_storage, d_gate, d_in, d_saved, d_grad_out, d_grad_gate, d_grad_in,
                 offsets_or_length, d_init=None, d_grad_last=None, d_grad_init=None, mode="sigmoid"):
        """Gradients of d_gate, d_in and d_init from those of d_out (None: zero) and d_last (None: zero); d_gate,
        d_in, d_saved and d_init are the Forward call's.  d_grad_init has one row per sequence, also for an
        expanded d_init (whose gradient is the sum of the rows).  d_grad_gate and d_grad_in may be d_gate, d_in or
        d_grad_out (with the same row stride), and d_grad_init may be d_init; other overlaps are refused."""
        if d_saved is None:
            raise ValueError("d_saved is needed: give it to Forward first")
        dt, gate = _float_dtype(d_gate, d_in, d_grad_out, d_grad_gate, d_grad_in), _gate(mode)
        offsets = offsets_or_length if isinstance(offsets_or_length, torch.Tensor) else None
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_gate, d_in, d_saved, d_grad_out, d_grad_gate, d_grad_in, d_init, d_grad_last, d_grad_init,
                temp_storage, offsets)
        _one_device(*keep)
        pg, sg, rows, channels = _matrix(d_gate, "d_gate")
        pi, si = _like(d_in, d_gate, rows, channels, "d_in")
        pgo, sgo = _like(d_grad_out, d_gate, rows, channels, "d_grad_out")
        pgg, sgg = _like(d_grad_gate, d_gate, rows, channels, "d_grad_gate")
        pgi, sgi = _like(d_grad_in, d_gate, rows, channels, "d_grad_in")
        count, length, off = self._sequences(offsets_or_length, rows)
        p0, s0 = self._init(d_init, count, channels)
        pgl = _dense(d_grad_last, (count, channels), _F32, "d_grad_last")
        pg0 = _dense(d_grad_init, (count, channels), _F32, "d_grad_init")
        self._call(cmdlist, L.lib().lcpp_linear_recurrence_backward,
                   (gate, dt, pg, sg, pi, si, _saved(d_saved, rows, channels), p0, s0, pgo, sgo, pgl, pgg, sgg, pgi,
                    sgi, pg0, rows, channels, count, length, off, temp, temp_bytes),
                   keep, "DeviceLinearRecurrence.Backward")

    def Step(self, cmdlist, d_gate, d_in, d_states_in, d_states_out, d_out=None, d_parents=None, mode="sigmoid"):
        """One token for each row: row i goes on from d_states_in[d_parents[i]] (without d_parents row i, a negative
        parent from zeros) to d_states_out[i], and d_out[i] is its rounding.  d_states_out may be d_states_in when
        there are no parents, and d_out may be d_gate or d_in (with the same row stride); other overlaps are
        refused."""
        dt, gate = _float_dtype(d_gate, d_in, d_out), _gate(mode)
        keep = (d_gate, d_in, d_states_in, d_states_out, d_out, d_parents)
        _one_device(*keep)
        pg, sg, rows, channels = _matrix(d_gate, "d_gate")
        pi, si = _like(d_in, d_gate, rows, channels, "d_in")
        po, so = _like(d_out, d_gate, rows, channels, "d_out")
        rows_in = 0 if d_states_in is None else d_states_in.shape[0]
        psi = _dense(d_states_in, (rows_in, channels), _F32, "d_states_in")
        pso = _dense(d_states_out, (rows, channels), _F32, "d_states_out")
        pp = _dense(d_parents, (rows,), _I32, "d_parents")
        self._call(cmdlist, L.lib().lcpp_linear_recurrence_step,
                   (gate, dt, pg, sg, pi, si, psi, rows_in, pp, pso, po, so, rows, channels),
                   keep, "DeviceLinearRecurrence.Step")


def _saved(d_saved, rows, channels):
    if d_saved is None:
        return None
    if not d_saved.is_contiguous():
        raise ValueError("d_saved must be contiguous")
    if _nbytes(d_saved) < DeviceLinearRecurrence.GetSavedStateBytes(rows, channels):
        raise ValueError("d_saved must hold GetSavedStateBytes(rows, channels) bytes")
    return d_saved.data_ptr()


class DeviceBeamSearch(_Recorded):
    """Selection of the best continuations of every batch entry's beams, and states that follow them."""

    @staticmethod
    def GetTempStorageBytes(num_batches: int, num_beams: int, vocab: int) -> int:
        return int(L.lib().lcpp_beam_select_temp_bytes(num_batches, num_beams, vocab))

    def Select(self, cmdlist, temp_storage, d_logits, d_scores, d_finished, d_scores_out, d_tokens_out,
               d_parents_out, d_finished_out, eos_token: int = -1):
        """d_logits: (batches * beams, vocab) or (batches, beams, vocab), any row stride; the other buffers
        (batches, beams).  Each beam offers its `beams` best tokens with d_scores + log_softmax(d_logits); the
        `beams` best of an entry come out, best first, with their token, their parent (a row of d_logits, for
        Reorder and DeviceLinearRecurrence.Step) and whether they are finished (d_finished of the parent, or
        the token eos_token).  A finished beam offers itself, with eos_token and its score.  d_finished and
        d_finished_out may be None.  Outputs that overlap an input or one another are refused."""
        dt = _float_dtype(d_logits)
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_logits, d_scores, d_finished, d_scores_out, d_tokens_out, d_parents_out, d_finished_out, temp_storage)
        _one_device(*keep)
        shape = d_scores.shape
        if len(shape) != 2:
            raise ValueError("d_scores must have the shape (batches, beams)")
        batches, beams = shape
        pz, sz, rows, vocab = _matrix(d_logits, "d_logits")
        if rows != batches * beams:
            raise ValueError("d_logits must have a row for each score")
        if not -0x80000000 <= eos_token <= 0x7fffffff:  # the entry's is 32 bits wide
            raise ValueError("eos_token must be a token (or negative: there is none)")
        pi, po = _dense(d_scores, shape, _F32, "d_scores"), _dense(d_scores_out, shape, _F32, "d_scores_out")
        pt, pp = _dense(d_tokens_out, shape, _I32, "d_tokens_out"), _dense(d_parents_out, shape, _I32, "d_parents_out")
        pf, pfo = _dense(d_finished, shape, _U8, "d_finished"), _dense(d_finished_out, shape, _U8, "d_finished_out")
        self._call(cmdlist, L.lib().lcpp_beam_select,
                   (dt, pz, sz, pi, pf, po, pt, pp, pfo, batches, beams, vocab, eos_token, temp, temp_bytes),
                   keep, "DeviceBeamSearch.Select")

    def Reorder(self, cmdlist, d_in, d_out, d_parents):
        """d_out[..., i, :] = d_in[..., d_parents[i], :] for states of any element type and the shape
        (rows, width) or (layers, rows, ...), the elements of a row adjacent; a negative parent gives zeros.
        d_out must not overlap d_in."""
        if d_in.dtype != d_out.dtype:
            raise TypeError("d_in and d_out must have the same element type")
        keep = (d_in, d_out, d_parents)
        _one_device(*keep)
        pi, li, ri, layers, rows_in, width = _layers(d_in, "d_in")
        po, lo, ro, layers_out, rows, width_out = _layers(d_out, "d_out")
        if layers_out != layers or width_out != width:
            raise ValueError("d_in and d_out must have the same layers and row shape")
        if d_parents.dtype != torch.int32 or d_parents.numel() != rows or not d_parents.is_contiguous():
            raise ValueError("d_parents must be a contiguous int32 tensor with one parent for each row of d_out")
        self._call(cmdlist, L.lib().lcpp_beam_reorder,
                   (pi, li, ri, po, lo, ro, d_parents.data_ptr(), layers, rows_in, rows, width),
                   keep, "DeviceBeamSearch.Reorder")


def _layers(t, name):
    """(pointer, layer stride, row stride, layers, rows, row bytes) of states, strides in bytes."""
    shape, stride, e = t.shape, t.stride(), t.element_size()
    if len(shape) == 3:  # the usual one
        layers, rows, width = shape
        outer, row, unit = stride
        if unit != 1 and width > 1:
            raise ValueError(f"{name}: the elements of a row must be adjacent")
        if row < width and rows > 1:
            raise ValueError(f"{name}: rows must not overlap")
        return t.data_ptr(), outer * e, row * e, layers, rows, width * e
    if len(shape) < 2:
        raise ValueError(f"{name} must have the shape (rows, width) or (layers, rows, ...)")
    if len(shape) == 2:
        shape, stride = (1, *shape), (0, *stride)
    width = 1
    for n, st in zip(shape[:1:-1], stride[:1:-1]):
        if n > 1 and st != width:
            raise ValueError(f"{name}: the elements of a row must be adjacent")
        width *= n
    if shape[1] > 1 and stride[1] < width:
        raise ValueError(f"{name}: rows must not overlap")
    return t.data_ptr(), stride[0] * e, stride[1] * e, shape[0], shape[1], width * e
