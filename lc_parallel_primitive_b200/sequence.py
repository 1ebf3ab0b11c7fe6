"""Operators over sequences, in the manner of the Device* classes: the gated
linear recurrence with its backward pass and single-token step
(DeviceLinearRecurrence), the gated delta rule, whose states are matrices,
likewise (DeviceDeltaRule), beam search's selection and reordering of states
(DeviceBeamSearch), and the cross entropy over a vocabulary from hidden states
with its gradients (DeviceCrossEntropy).

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


class DeviceDeltaRule(_Recorded):
    """Gated delta rule: per sequence and head a state S (value_dim, key_dim), and for each token

        S' = exp(decay) S,  u = beta (v - S' k),  S = S' + u k^T,  out = scale S q

    d_q, d_k: (rows, key_heads, key_dim) or (batch, time, key_heads, key_dim), d_v and d_out the same with heads and
    value_dim; heads of a row adjacent, any row stride; head h reads key head h // (heads // key_heads).  d_decay (log
    of the factor, <= 0; None: 0) and d_beta: float32 (rows, heads), any row stride.  Dimensions up to 128.  scale:
    None for 1 / sqrt(key_dim).  offsets_or_length as in DeviceLinearRecurrence; states are contiguous float32
    (sequences, heads, value_dim, key_dim).  temp_storage is contiguous and 16-byte aligned, as temp_buffer's is.
    Inputs are finite: the work goes by 64 rows and 16 value dimensions, so a NaN reaches up to 63 rows of its sequence
    before it and value dimensions beside it, too, but no other sequence or head.  float32 values enter products in two
    float16 parts, bf16 outputs are made of 11 bits of the state; include/lcpp_b200.h states precision and range.
    """

    @staticmethod
    def _shape(num_rows, num_sequences, heads, key_heads, key_dim, value_dim, length=0, offsets=None, scale=0.0):
        return L.DeltaShape(num_rows, num_sequences, length, offsets, heads, key_heads, key_dim, value_dim, scale)

    @staticmethod
    def GetTempStorageBytes(num_rows: int, num_sequences: int, heads: int, key_heads: int, key_dim: int, value_dim: int,
                            dtype=torch.bfloat16, backward: bool = True) -> int:
        """For Forward, or (backward) for both calls, with so many rows and sequences or fewer."""
        if dtype not in _FLOATS:
            raise TypeError(f"unsupported element type {dtype}")
        shape = DeviceDeltaRule._shape(num_rows, num_sequences, heads, key_heads, key_dim, value_dim)
        return int(L.lib().lcpp_delta_rule_temp_bytes(_FLOATS[dtype], shape, backward))

    @staticmethod
    def GetSavedStateBytes(num_rows: int, num_sequences: int, heads: int, key_heads: int, key_dim: int, value_dim: int) -> int:
        """Bytes of d_saved, which Forward fills for Backward; for so many rows and sequences or fewer."""
        shape = DeviceDeltaRule._shape(num_rows, num_sequences, heads, key_heads, key_dim, value_dim)
        return int(L.lib().lcpp_delta_rule_saved_bytes(shape))

    @staticmethod
    def _inputs(d_q, d_k, d_v, d_decay, d_beta):
        """(inputs without states, rows, heads, key_heads, key_dim, value_dim)."""
        pq, sq, rows, key_heads, key_dim = _heads(d_q, "d_q")
        pk, sk, rk, hk, dk = _heads(d_k, "d_k")
        pv, sv, rv, heads, value_dim = _heads(d_v, "d_v")
        if rk != rows or hk != key_heads or dk != key_dim:
            raise ValueError("d_q and d_k must have the same shape")
        if rv != rows:
            raise ValueError("d_v must have the rows of d_q")
        if not key_heads or heads % key_heads:
            raise ValueError(f"{heads} heads are no whole number for each of {key_heads} key heads")
        if key_dim > 128 or value_dim > 128 or not key_dim or not value_dim:
            raise ValueError("key_dim and value_dim must be from 1 to 128")
        pb, sb = _gates(d_beta, rows, heads)
        pd, sd = (None, 0) if d_decay is None else _gates(d_decay, rows, heads)
        return L.DeltaInputs(pq, pk, pv, sq, sk, sv, pd, pb, sd, sb, None), rows, heads, key_heads, key_dim, value_dim

    def _sequences(self, inputs, offsets_or_length, rows, heads, key_heads, key_dim, value_dim, d_init, scale):
        """(shape, shape of the states)."""
        count, length, off = DeviceLinearRecurrence._sequences(offsets_or_length, rows)
        states = (count, heads, value_dim, key_dim)
        inputs.init = _dense(d_init, states, _F32, "d_init")
        if scale is None:
            scale = key_dim ** -0.5
        return self._shape(rows, count, heads, key_heads, key_dim, value_dim, length, off, scale), states

    def Forward(self, cmdlist, temp_storage, d_q, d_k, d_v, d_decay, d_beta, d_out, offsets_or_length, d_init=None,
                d_last=None, d_saved=None, scale=None):
        """d_out, and d_last = the states after each sequence's last row (d_init for an empty sequence).  d_last may be
        d_init; other overlaps are refused."""
        dt = _float_dtype(d_q, d_k, d_v, d_out)
        offsets = offsets_or_length if isinstance(offsets_or_length, torch.Tensor) else None
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_q, d_k, d_v, d_decay, d_beta, d_out, d_init, d_last, d_saved, temp_storage, offsets)
        _one_device(*keep)
        inputs, *sizes = self._inputs(d_q, d_k, d_v, d_decay, d_beta)
        shape, states = self._sequences(inputs, offsets_or_length, *sizes, d_init, scale)
        po, so, *like = _heads(d_out, "d_out")
        if like != [sizes[0], sizes[1], sizes[4]]:
            raise ValueError("d_out must have the shape of d_v")
        pl = _dense(d_last, states, _F32, "d_last")
        self._call(cmdlist, L.lib().lcpp_delta_rule_forward,
                   (dt, shape, inputs, po, so, pl, self._saved(d_saved, shape), temp, temp_bytes),
                   keep, "DeviceDeltaRule.Forward")

    @staticmethod
    def _saved(d_saved, shape):
        if d_saved is None:
            return None
        if not d_saved.is_contiguous():
            raise ValueError("d_saved must be contiguous")
        if _nbytes(d_saved) < L.lib().lcpp_delta_rule_saved_bytes(shape):
            raise ValueError("d_saved must hold GetSavedStateBytes(...) bytes")
        return d_saved.data_ptr()

    def Backward(self, cmdlist, temp_storage, d_q, d_k, d_v, d_decay, d_beta, d_saved, d_grad_out, d_grad_q, d_grad_k,
                 d_grad_v, d_grad_decay, d_grad_beta, offsets_or_length, d_init=None, d_grad_last=None, d_grad_init=None,
                 scale=None):
        """Gradients of the inputs from those of d_out (None: zero) and d_last (None: zero); the inputs, d_init, scale
        and d_saved are the Forward call's.  Gradients are contiguous, of the inputs' shapes and types; d_grad_decay
        and d_grad_init may be None.  Outputs must not overlap anything else."""
        if d_saved is None:
            raise ValueError("d_saved is needed: give it to Forward first")
        dt = _float_dtype(d_q, d_k, d_v, d_grad_out, d_grad_q, d_grad_k, d_grad_v)
        offsets = offsets_or_length if isinstance(offsets_or_length, torch.Tensor) else None
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_q, d_k, d_v, d_decay, d_beta, d_saved, d_grad_out, d_grad_q, d_grad_k, d_grad_v, d_grad_decay,
                d_grad_beta, d_init, d_grad_last, d_grad_init, temp_storage, offsets)
        _one_device(*keep)
        inputs, *sizes = self._inputs(d_q, d_k, d_v, d_decay, d_beta)
        shape, states = self._sequences(inputs, offsets_or_length, *sizes, d_init, scale)
        pgo, sgo = None, 0
        if d_grad_out is not None:
            pgo, sgo, *like = _heads(d_grad_out, "d_grad_out")
            if like != [sizes[0], sizes[1], sizes[4]]:
                raise ValueError("d_grad_out must have the shape of d_v")
        own = (d_q.dtype,)
        grads = L.DeltaGrads(pgo, sgo, _dense(d_grad_last, states, _F32, "d_grad_last"),
                             _dense(d_grad_q, d_q.shape, own, "d_grad_q"), _dense(d_grad_k, d_k.shape, own, "d_grad_k"),
                             _dense(d_grad_v, d_v.shape, own, "d_grad_v"),
                             _dense(d_grad_decay, d_beta.shape, _F32, "d_grad_decay"),
                             _dense(d_grad_beta, d_beta.shape, _F32, "d_grad_beta"),
                             _dense(d_grad_init, states, _F32, "d_grad_init"))
        self._call(cmdlist, L.lib().lcpp_delta_rule_backward,
                   (dt, shape, inputs, self._saved(d_saved, shape), grads, temp, temp_bytes),
                   keep, "DeviceDeltaRule.Backward")

    def Step(self, cmdlist, d_q, d_k, d_v, d_decay, d_beta, d_states_in, d_states_out, d_out, d_parents=None, scale=None):
        """One token for each row: row i goes on from d_states_in[d_parents[i]] (without d_parents row i; a negative
        parent, or d_states_in None, from zeros) to d_states_out[i] (rows, heads, value_dim, key_dim).  d_states_out may
        be d_states_in when there are no parents; other overlaps are refused."""
        dt = _float_dtype(d_q, d_k, d_v, d_out)
        keep = (d_q, d_k, d_v, d_decay, d_beta, d_states_in, d_states_out, d_out, d_parents)
        _one_device(*keep)
        usual = self._usual_step(d_q, d_k, d_v, d_decay, d_beta, d_states_in, d_states_out, d_out)
        if usual is not None:
            inputs, rows, heads, key_heads, key_dim, value_dim, rows_in, pn, po = usual
            so = heads * value_dim
        else:
            inputs, rows, heads, key_heads, key_dim, value_dim = self._inputs(d_q, d_k, d_v, d_decay, d_beta)
            state = (heads, value_dim, key_dim)
            rows_in = 0
            if d_states_in is not None:
                rows_in = d_states_in.shape[0]
                inputs.init = _dense(d_states_in, (rows_in, *state), _F32, "d_states_in")
            pn = _dense(d_states_out, (rows, *state), _F32, "d_states_out")
            po, so, r, h, d = _heads(d_out, "d_out")
            if r != rows or h != heads or d != value_dim:
                raise ValueError("d_out must have the shape of d_v")
        pp = _dense(d_parents, (rows,), _I32, "d_parents")
        if scale is None:
            scale = key_dim ** -0.5
        shape = L.DeltaShape(rows, 0, 0, None, heads, key_heads, key_dim, value_dim, scale)
        self._call(cmdlist, L.lib().lcpp_delta_rule_step, (dt, shape, inputs, rows_in, pp, pn, po, so), keep,
                   "DeviceDeltaRule.Step")

    @staticmethod
    def _usual_step(d_q, d_k, d_v, d_decay, d_beta, d_states_in, d_states_out, d_out):
        """What Step passes on, for contiguous tensors of the shapes (rows, ...) that all fit; else None."""
        q, v, n = d_q.shape, d_v.shape, d_states_out.shape
        if len(q) != 3 or len(v) != 3 or len(n) != 4 or d_states_in is None or d_decay is None:
            return None
        rows, key_heads, key_dim = q
        r, heads, value_dim = v
        gates = d_beta.shape
        before = d_states_in.shape
        if (r != rows or d_k.shape != q or d_out.shape != v or not 0 < key_dim <= 128 or not 0 < value_dim <= 128 or not key_heads
                or heads % key_heads or len(gates) != 2 or gates[0] != rows or gates[1] != heads or d_decay.shape != gates
                or n[0] != rows or n[1] != heads or n[2] != value_dim or n[3] != key_dim or before[1:] != n[1:]):
            return None
        f32 = torch.float32
        if d_decay.dtype != f32 or d_beta.dtype != f32 or d_states_in.dtype != f32 or d_states_out.dtype != f32:
            return None
        if not (d_q.is_contiguous() and d_k.is_contiguous() and d_v.is_contiguous() and d_decay.is_contiguous()
                and d_beta.is_contiguous() and d_states_in.is_contiguous() and d_states_out.is_contiguous() and d_out.is_contiguous()):
            return None
        keys, values = key_heads * key_dim, heads * value_dim
        return (L.DeltaInputs(d_q.data_ptr(), d_k.data_ptr(), d_v.data_ptr(), keys, keys, values, d_decay.data_ptr(), d_beta.data_ptr(),
                              heads, heads, d_states_in.data_ptr()),
                rows, heads, key_heads, key_dim, value_dim, before[0], d_states_out.data_ptr(), d_out.data_ptr())


def _gates(t, rows, heads):
    """(pointer, row stride) of decays or strengths."""
    if t.dtype != torch.float32:
        raise TypeError("d_decay and d_beta must have the element type torch.float32")
    shape = t.shape
    if len(shape) == 2 and shape[0] == rows and shape[1] == heads and t.is_contiguous():  # the usual one
        return t.data_ptr(), heads
    pointer, row, r, h = _matrix(t, "d_decay and d_beta")
    if r != rows or h != heads:
        raise ValueError(f"d_decay and d_beta must have the shape {(rows, heads)}")
    return pointer, row


def _heads(t, name):
    """(pointer, row stride, rows, heads, dim) of a (rows, heads, dim) or (batch, time, heads, dim) tensor whose rows are
    one stride apart and whose heads are adjacent."""
    shape = t.shape
    if len(shape) == 3 and t.is_contiguous():  # the usual one
        rows, heads, dim = shape
        return t.data_ptr(), heads * dim, rows, heads, dim
    stride = t.stride()
    if len(shape) == 4:
        batch, time, heads, dim = shape
        rows, row = batch * time, stride[1]
        if time == 1:
            row = stride[0]
        elif batch > 1 and rows and stride[0] != time * row:
            raise ValueError(f"{name}: the batch stride must be the row stride times the length")
    elif len(shape) == 3:
        rows, heads, dim = shape
        row = stride[0]
    else:
        raise ValueError(f"{name} must have the shape (rows, heads, dim) or (batch, time, heads, dim)")
    if rows and ((dim > 1 and stride[-1] != 1) or (heads > 1 and stride[-2] != dim)):
        raise ValueError(f"{name}: the heads of a row must be adjacent")
    if row < heads * dim and rows > 1:
        raise ValueError(f"{name}: rows must not overlap")
    return t.data_ptr(), row, rows, heads, dim


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


class DeviceCrossEntropy(_Recorded):
    """Softmax cross entropy over a vocabulary from hidden states, without the logits in memory.

    loss[i] = log sum_v exp(z_iv) - z_i,target(i) with z = d_hidden d_weight^T.  d_hidden: (rows, channels) or
    (batch, time, channels), any row stride; d_weight: (vocab, channels) of the same type; d_targets: int32, one for
    each row.  A row with a negative target takes no part: loss, logsum and gradient 0, whatever its hidden state
    holds.  Sums are float32; float32 operands are multiplied in two float16 or three bf16 parts.
    """

    @staticmethod
    def GetTempStorageBytes(num_rows: int, num_channels: int, vocab: int, dtype=torch.bfloat16, backward: bool = True,
                            aligned: bool = True) -> int:
        """For Forward, or for both calls, with so many rows or fewer; aligned=False: rows of d_weight may start off a
        16-byte boundary."""
        if dtype not in _FLOATS:
            raise TypeError(f"unsupported element type {dtype}")
        return int(L.lib().lcpp_cross_entropy_temp_bytes(_FLOATS[dtype], num_rows, num_channels, vocab, backward, aligned))

    @staticmethod
    def _operands(d_hidden, d_weight, d_targets):
        """(hidden pointer, stride, weight pointer, stride, targets pointer, rows, channels, vocab)."""
        ph, sh, rows, channels = _matrix(d_hidden, "d_hidden")
        if d_weight.dim() != 2 or d_weight.shape[1] != channels:
            raise ValueError(f"d_weight must have the shape (vocab, {channels}), not {tuple(d_weight.shape)}")
        pw, sw, vocab, _ = _matrix(d_weight, "d_weight")
        if d_targets.dtype != torch.int32:
            raise TypeError("d_targets must have the element type torch.int32")
        if d_targets.numel() != rows or not d_targets.is_contiguous():
            raise ValueError("d_targets must be contiguous, one for each row of d_hidden")
        return ph, sh, pw, sw, d_targets.data_ptr(), rows, channels, vocab

    def Forward(self, cmdlist, temp_storage, d_hidden, d_weight, d_targets, d_loss, d_logsum=None):
        """d_loss and d_logsum (for Backward): float32, one for each row; either may be None."""
        dt = _float_dtype(d_hidden, d_weight)
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_hidden, d_weight, d_targets, d_loss, d_logsum, temp_storage)
        _one_device(*keep)
        ph, sh, pw, sw, pt, rows, channels, vocab = self._operands(d_hidden, d_weight, d_targets)
        pl, ps = _per_row(d_loss, rows, "d_loss"), _per_row(d_logsum, rows, "d_logsum")
        self._call(cmdlist, L.lib().lcpp_cross_entropy_forward,
                   (dt, ph, sh, pw, sw, pt, pl, ps, rows, channels, vocab, temp, temp_bytes),
                   keep, "DeviceCrossEntropy.Forward")

    def Backward(self, cmdlist, temp_storage, d_hidden, d_weight, d_targets, d_logsum, d_grad_loss, d_grad_hidden,
                 d_grad_weight):
        """Gradients of d_hidden and d_weight (None: not wanted) from that of the loss: float32, one for each row, or
        one expanded over the rows (stride 0); d_logsum is the Forward call's.  Outputs must not overlap anything
        else."""
        dt = _float_dtype(d_hidden, d_weight, d_grad_hidden, d_grad_weight)
        temp, temp_bytes = _temp(temp_storage)
        keep = (d_hidden, d_weight, d_targets, d_logsum, d_grad_loss, d_grad_hidden, d_grad_weight, temp_storage)
        _one_device(*keep)
        ph, sh, pw, sw, pt, rows, channels, vocab = self._operands(d_hidden, d_weight, d_targets)
        ps = _per_row(d_logsum, rows, "d_logsum")
        if d_grad_loss.dtype != torch.float32:
            raise TypeError("d_grad_loss must have the element type torch.float32")
        if d_grad_loss.numel() != rows:
            raise ValueError("d_grad_loss must hold one value for each row")
        one = rows > 0 and all(n == 1 or st == 0 for n, st in zip(d_grad_loss.shape, d_grad_loss.stride()))
        if not one and not d_grad_loss.is_contiguous():
            raise ValueError("d_grad_loss must be contiguous or one value expanded")
        pgh, sgh = _like(d_grad_hidden, d_hidden, rows, channels, "d_grad_hidden")
        pgw, sgw = _like(d_grad_weight, d_weight, vocab, channels, "d_grad_weight")
        self._call(cmdlist, L.lib().lcpp_cross_entropy_backward,
                   (dt, ph, sh, pw, sw, pt, ps, d_grad_loss.data_ptr(), 0 if one else 1, pgh, sgh, pgw, sgw, rows,
                    channels, vocab, temp, temp_bytes),
                   keep, "DeviceCrossEntropy.Backward")


def _per_row(t, rows, name):
    """Pointer of a contiguous float32 tensor with one value for each row (None stays None)."""
    if t is None:
        return None
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must have the element type torch.float32")
    if t.numel() != rows or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous, one value for each row")
    return t.data_ptr()


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
