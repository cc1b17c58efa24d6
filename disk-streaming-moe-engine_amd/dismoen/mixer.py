"""The token mixer of the port block's linear-attention layers over libdismoen_hip.so.

Between the mixer's two projections (src/layers/port_scheduler.mojo:286-372):
  ShortConv        causal depthwise convolution with a state per sequence
  GatedDelta       the gated delta rule with a state per sequence
  GatedNorm        norms after and before a block, with its gate and residual
  GatedDeltaMixer  the three together, as a layer runs them
A SeqBatch says which rows are which sequence's.  An operator is made once per
layer, with its weights, and called once per step.

Arrays are torch tensors on the block's device (the call is queued on the
block's stream and returns at once; errors in the sequences are reported by
MoEBlock.sync()), or numpy arrays, all of them (the call is synchronous; bf16
rows are their uint16 bit patterns).  Outputs are arrays of the caller's.  A
block's stream is its own: order work of other streams against it, or give it
theirs (MoEBlock.set_stream).  PortBlock does so for torch's current stream.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np

from ._lib import (DMH_F_CHECK, DMH_F_DEVICE, DismoenError, DmhGatedDelta, DmhGatedNorm, DmhSeqBatch,
                   DmhShortConv, check, errbuf)

F32, F16, BF16 = 0, 1, 2
GATES = {None: 0, "silu": 1, "sigmoid": 2}
_WRITTEN = ("out", "stream", "y")  # the names of row arrays that a call writes
_TYPES = {np.dtype(np.float32): F32, np.dtype(np.float16): F16, np.dtype(np.uint16): BF16}


def _type(a) -> int:
    t = _TYPES.get(a.dtype)
    if t is None and not isinstance(a, np.ndarray) and len(_TYPES) == 3:
        import torch
        _TYPES.update({torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16})
        t = _TYPES.get(a.dtype)
    if t is None:
        raise _bad(f"rows are float32, float16 or bfloat16, not {a.dtype}")
    return t


def _bad(text: str) -> DismoenError:
    return DismoenError(1, '{"error_type":"CONFIG_ERROR","detail":"' + text + '","stage":"mixer"}')


def _strides(a):
    return tuple(s // a.itemsize for s in a.strides) if isinstance(a, np.ndarray) else a.stride()


def _packed(shape, strides) -> bool:
    """Whether the elements of these dimensions lie one behind the other."""
    want = 1
    for n, s in zip(reversed(shape), reversed(strides)):
        if n != 1 and s != want:
            return False
        want *= n
    return True


class _Operator:
    """A call's argument block, filled field by field; checks that all of its
    arrays are on one side, the host's (device None) or the block's device."""

    def __init__(self, blk):
        self._blk = blk
        self._err = errbuf()
        self._sides = set()
        self._kept = []

    def _weight(self, a, shape, what):
        """The address of an fp32 weight that the operator keeps."""
        if a is None:
            return None
        if tuple(a.shape) != shape or _type(a) != F32 or not _packed(a.shape, _strides(a)):
            raise _bad(f"{what} must be a contiguous float32 array of shape {list(shape)}")
        host = isinstance(a, np.ndarray)
        if not host and a.get_device() != self._blk.device:
            raise _bad(f"{what} must be on the block's device, cuda:{self._blk.device}")
        self._kept.append(a)
        self._sides.add(host)
        if len(self._sides) > 1:
            raise _bad("numpy arrays and device tensors in one operator")
        return a.ctypes.data if host else a.data_ptr()

    def _side(self, a):
        """Whether the call's arrays are the host's, as `a` and the weights are."""
        host = isinstance(a, np.ndarray)
        if self._sides and host not in self._sides:
            raise _bad("numpy arrays and device tensors in one call")
        return host

    # (called for each array of each call: no more Python than it takes)
    def _rows(self, a, heads, dim, dtype, device, what):
        """(rows, address, stride) of a row array [rows][heads][dim]."""
        if device is None:
            if not isinstance(a, np.ndarray) or a.ndim != 3:
                raise _bad(f"{what} must be a numpy array as the others, [rows][{heads}][{dim}]")
            if what in _WRITTEN and not a.flags.writeable:
                raise _bad(f"{what} is written, and the array is read-only")
            (n, h, d), (s, sh, sd), p = a.shape, _strides(a), a.ctypes.data
        else:
            try:
                n, h, d = a.shape
                s, sh, sd = a.stride()
                if a.get_device() != device:
                    raise ValueError
            except (ValueError, AttributeError, TypeError):
                raise _bad(f"{what} must be a tensor on cuda:{device}, [rows][{heads}][{dim}]") \
                    from None
            p = a.data_ptr()
        if h != heads or d != dim or a.dtype != dtype or (sd != 1 and d != 1) \
                or (sh != d and h != 1):
            raise _bad(f"{what} must be rows of {heads} times {dim} elements, packed, of the"
                       " call's type")
        return n, p, s if n > 1 else max(s, h * d)

    def _rows1(self, a, dim, dtype, device, what):
        """The same of [rows][dim]."""
        if device is None:
            if not isinstance(a, np.ndarray) or a.ndim != 2:
                raise _bad(f"{what} must be a numpy array as the others, [rows][{dim}]")
            if what in _WRITTEN and not a.flags.writeable:
                raise _bad(f"{what} is written, and the array is read-only")
            (n, d), (s, sd), p = a.shape, _strides(a), a.ctypes.data
        else:
            try:
                n, d = a.shape
                s, sd = a.stride()
                if a.get_device() != device:
                    raise ValueError
            except (ValueError, AttributeError, TypeError):
                raise _bad(f"{what} must be a tensor on cuda:{device}, [rows][{dim}]") from None
            p = a.data_ptr()
        if d != dim or a.dtype != dtype or (sd != 1 and d != 1):
            raise _bad(f"{what} must be rows of {dim} elements, packed, of the call's type")
        return n, p, s if n > 1 else max(s, d)

    def _state(self, a, shape, dtype, device, batch):
        host = isinstance(a, np.ndarray)
        if host is not (device is None) or a.shape != (batch.num_slots, *shape) \
                or _type(a) != dtype or not (a.flags.c_contiguous if host else a.is_contiguous()) \
                or (not host and a.get_device() != device):
            raise _bad(f"state must be a contiguous array [num_slots]{list(shape)}")
        if host and not a.flags.writeable:
            raise _bad("state is written, and the array is read-only")
        if batch.device != device:
            raise _bad("the batch's arrays are not where the call's are")
        return a.ctypes.data if host else a.data_ptr()


class SeqBatch:
    """The sequences of a step: rows offsets[i] .. offsets[i + 1] - 1 are sequence
    i's, its state is state slots[i] (None: i; negative: the sequence is
    skipped), and one marked in `fresh` starts from zeros.  offsets, slots and
    fresh are int32, torch tensors or numpy arrays; total_tokens and max_len
    bound the rows and any sequence's length.  The arrays are read by each call,
    so their values may change between steps."""

    def __init__(self, offsets, total_tokens: int, max_len: int, num_slots: int, slots=None,
                 fresh=None):
        n = offsets.shape[0] - 1
        self.total_tokens, self.num_slots = int(total_tokens), int(num_slots)
        if not all(0 <= v < 1 << 31 for v in (n, self.total_tokens, self.num_slots, int(max_len))):
            raise _bad("total_tokens, max_len, num_slots and the number of sequences are int32"
                       " values from 0 on")
        self.host = isinstance(offsets, np.ndarray)
        self.device = None if self.host else offsets.get_device()
        self.arrays = (offsets, slots, fresh)
        ptrs = []
        for a, want, what in ((offsets, n + 1, "offsets"), (slots, n, "slots"),
                              (fresh, n, "fresh")):
            if a is None:
                ptrs.append(None)
                continue
            if isinstance(a, np.ndarray) is not self.host or a.ndim != 1 or a.shape[0] != want \
                    or str(a.dtype).split(".")[-1] != "int32" or not _packed(a.shape, _strides(a)):
                raise _bad(f"{what} must be {want} int32 values on the side of offsets")
            if not self.host and (not a.is_cuda or a.get_device() != self.device):
                raise _bad(f"{what} must be on the device")
            ptrs.append(a.ctypes.data if self.host else a.data_ptr())
        self._c = DmhSeqBatch(n, self.total_tokens, int(max_len), self.num_slots, *ptrs)
        self._ref = C.addressof(self._c)


class ShortConv(_Operator):
    """Causal depthwise convolution: weight [channels][width] and bias [channels]
    fp32, SiLU where `silu`."""

    def __init__(self, blk, weight, bias=None, silu: bool = True):
        super().__init__(blk)
        if weight.ndim != 2:
            raise _bad("weight must be [channels][width]")
        self.channels, self.width = weight.shape
        a = self._c = DmhShortConv()
        a.channels, a.width, a.silu = self.channels, self.width, int(silu)
        a.weight = self._weight(weight, (self.channels, self.width), "weight")
        a.bias = self._weight(bias, (self.channels,), "bias")
        self._ref = C.addressof(a)

    def __call__(self, x, state, batch: SeqBatch, out):
        """out[t] for the rows x [rows][channels]; state [num_slots][width - 1]
        [channels], the last rows of each sequence, is brought up to date."""
        self._go(batch, self._set(x, state, batch, out))
        return out

    def _set(self, x, state, batch, out):
        """Fills the argument block from the arrays, which it checks; the call's flags."""
        c, t, w = self._c, x.dtype, self.channels
        dev = None if self._side(x) else self._blk.device
        c.dtype = code = _type(x)
        nx, c.x, c.x_stride = self._rows1(x, w, t, dev, "x")
        ny, c.y, c.y_stride = self._rows1(out, w, t, dev, "out")
        c.state = self._state(state, (self.width - 1, w), code, dev, batch)
        if min(nx, ny) < batch.total_tokens:
            raise _bad("x or out has fewer rows than total_tokens")
        return 0 if dev is None else DMH_F_DEVICE

    def _go(self, batch, flags):
        blk, e = self._blk, self._err
        rc = blk._lib.dmh_short_conv_forward(blk.handle, self._ref, batch._ref, flags, e, 2048)
        if rc:
            check(rc, e)


class GatedDelta(_Operator):
    """The gated delta rule on v_heads heads (v_heads / k_heads of them share a
    key head).  With a_log [v_heads] the gates come raw: log decay =
    -exp(a_log) softplus(a + dt_bias), beta = sigmoid(b); without it a is the log
    decay and b is beta, in fp32.  scale: None is k_dim ** -0.5."""

    def __init__(self, blk, k_heads: int, v_heads: int, k_dim: int, v_dim: int, a_log=None,
                 dt_bias=None, qk_norm: bool = True, eps: float = 1e-6, scale: float | None = None):
        super().__init__(blk)
        a = self._c = DmhGatedDelta()
        a.k_heads, a.v_heads, a.k_dim, a.v_dim = k_heads, v_heads, k_dim, v_dim
        a.qk_norm, a.eps = int(qk_norm), eps
        a.scale = k_dim ** -0.5 if scale is None else scale
        a.a_log = self._weight(a_log, (v_heads,), "a_log")
        a.dt_bias = self._weight(dt_bias, (v_heads,), "dt_bias")
        self._raw = a_log is not None
        self._s = (v_heads, k_dim, v_dim)
        self._ref = C.addressof(a)

    def __call__(self, q, k, v, a, b, state, batch: SeqBatch, out):
        """out[t] [v_heads][v_dim] for rows q, k [rows][k_heads][k_dim], v
        [rows][v_heads][v_dim] and gates a, b [rows][v_heads]; state [num_slots]
        [v_heads][k_dim][v_dim] fp32 is brought up to date."""
        self._go(batch, self._set(q, k, v, a, b, state, batch, out))
        return out

    def _set(self, q, k, v, a, b, state, batch, out):
        c, t = self._c, v.dtype
        dev = None if self._side(v) else self._blk.device
        c.dtype = _type(v)
        g = t if self._raw else a.dtype
        if not self._raw and _type(a) != F32:
            raise _bad("without a_log, a and b must be float32")
        hk, hv, dk, dv = c.k_heads, c.v_heads, c.k_dim, c.v_dim
        rows = self._rows
        nq, c.q, c.q_stride = rows(q, hk, dk, t, dev, "q")
        nk, c.k, c.k_stride = rows(k, hk, dk, t, dev, "k")
        nv, c.v, c.v_stride = rows(v, hv, dv, t, dev, "v")
        na, c.a, c.a_stride = self._rows1(a, hv, g, dev, "a")
        nb, c.b, c.b_stride = self._rows1(b, hv, g, dev, "b")
        no, c.o, c.o_stride = rows(out, hv, dv, t, dev, "out")
        c.state = self._state(state, self._s, F32, dev, batch)
        if min(nq, nk, nv, na, nb, no) < batch.total_tokens:
            raise _bad("a row array has fewer rows than total_tokens")
        return 0 if dev is None else DMH_F_DEVICE

    def _go(self, batch, flags):
        blk, e = self._blk, self._err
        rc = blk._lib.dmh_gated_delta_forward(blk.handle, self._ref, batch._ref, flags, e, 2048)
        if rc:
            check(rc, e)


class GatedNorm(_Operator):
    """Norms after and before a block with its gate and residual, over rows of
    `groups` groups of `dim`:
      u      = rmsnorm(x) * gamma where `post`, else x; times silu or sigmoid of the gate
      stream = residual + scale * u      (scale: a number, or [groups][dim])
      y      = rmsnorm(stream) * edge_gamma where `edge`"""

    def __init__(self, blk, dim: int, groups: int = 1, gamma=None, edge_gamma=None,
                 post: bool = True, edge: bool = False, gate: str | None = None, scale=1.0,
                 eps: float = 1e-6):
        super().__init__(blk)
        if gate not in GATES:
            raise _bad("gate must be None, silu or sigmoid")
        if (gamma is not None and not post) or (edge_gamma is not None and not edge):
            raise _bad("gamma without post, or edge_gamma without edge")
        a = self._c = DmhGatedNorm()
        a.groups, a.dim, a.post, a.gate_act, a.eps = groups, dim, int(post), GATES[gate], eps
        a.gamma = self._weight(gamma, (dim,), "gamma")
        a.edge_gamma = self._weight(edge_gamma, (dim,), "edge_gamma")
        if isinstance(scale, (int, float)):
            a.scale = scale
        else:
            a.scale = 1.0
            a.scale_vec = self._weight(scale, (groups, dim), "scale")
        self._shape, self._edge, self._gate = (groups, dim), edge, gate is not None
        self._ref = C.addressof(a)

    def __call__(self, x, stream=None, y=None, gate=None, residual=None):
        """Writes stream and (where `edge`) y, arrays of the rows' shape [rows]
        [groups][dim]; stream may be the residual itself."""
        self._go(self._set(x, stream, y, gate, residual))
        return stream, y

    def _set(self, x, stream, y, gate, residual):
        if (gate is None) == self._gate or (y is None) == self._edge:
            raise _bad("gate and y are given exactly where the operator has them")
        out = y if stream is None else stream
        if out is None:
            raise _bad("neither stream nor y is given")
        c, t, so = self._c, x.dtype, out.dtype
        dev = None if self._side(x) else self._blk.device
        c.dtype, c.stream_dtype = _type(x), _type(out)
        h, d = self._shape
        rows = self._rows
        n, c.x, c.x_stride = rows(x, h, d, t, dev, "x")
        c.rows = m = n
        if gate is not None:
            m, c.gate, c.gate_stride = rows(gate, h, d, t, dev, "gate")
        if residual is not None:
            k, c.residual, c.residual_stride = rows(residual, h, d, so, dev, "residual")
            m = m if k == n else k
        else:
            c.residual = None
        if stream is not None:
            k, c.stream, c.stream_stride = rows(stream, h, d, so, dev, "stream")
            m = m if k == n else k
        else:
            c.stream = None
        if y is not None:
            k, c.y, c.y_stride = rows(y, h, d, so, dev, "y")
            m = m if k == n else k
        if m != n or n >= 1 << 31:
            raise _bad("the row arrays differ in their rows, or have 2^31 or more")
        return 0 if dev is None else DMH_F_DEVICE

    def _go(self, flags):
        blk, e = self._blk, self._err
        rc = blk._lib.dmh_gated_norm_forward(blk.handle, self._ref, flags, e, 2048)
        if rc:
            check(rc, e)


class GatedDeltaMixer:
    """One linear-attention layer between its projections: the convolution over
    the mixed rows [q | k | v], the gated delta rule, and the norm of each head's
    output, gated by silu(z).  conv_state [num_slots][width - 1][channels] and
    state [num_slots][v_heads][k_dim][v_dim] belong to the caller."""

    def __init__(self, blk, k_heads: int, v_heads: int, k_dim: int, v_dim: int, conv_weight,
                 a_log, dt_bias, norm_gamma, conv_bias=None, eps: float = 1e-6):
        self.channels = 2 * k_heads * k_dim + v_heads * v_dim
        self.k, self.v = (k_heads, k_dim), (v_heads, v_dim)
        self.conv = ShortConv(blk, conv_weight, bias=conv_bias)
        if self.conv.channels != self.channels:
            raise _bad(f"conv_weight must have {self.channels} channels")
        self.delta = GatedDelta(blk, k_heads, v_heads, k_dim, v_dim, a_log=a_log, dt_bias=dt_bias,
                                eps=eps)
        self.norm = GatedNorm(blk, v_dim, v_heads, gamma=norm_gamma, gate="silu", eps=eps)

    def __call__(self, mixed, z, b, a, conv_state, state, batch: SeqBatch, work, out):
        """out [rows][v_heads][v_dim], the input of the output projection, from the
        input projection's rows mixed [rows][channels], z [rows][v_heads][v_dim]
        and b, a [rows][v_heads].  work: rows like mixed, overwritten.  What out
        holds in rows of no sequence has no meaning.  A call that is refused leaves
        both states as they were."""
        n, kw = batch.total_tokens, self.k[0] * self.k[1]
        work, out = work[:n], out[:n]
        flags = self.conv._set(mixed, conv_state, batch, work)
        if isinstance(work, np.ndarray):
            q, k, v = (np.lib.stride_tricks.as_strided(
                work[:, at:], (n, *s), (work.strides[0], s[1] * work.itemsize, work.itemsize))
                for at, s in ((0, self.k), (kw, self.k), (2 * kw, self.v)))
        else:
            q, k, v = (work[:, at:at + s[0] * s[1]].unflatten(1, s)
                       for at, s in ((0, self.k), (kw, self.k), (2 * kw, self.v)))
        self.delta._set(q, k, v, a, b, state, batch, out)
        self.norm._set(out, out, None, z[:n], None)
        # (all that the library can refuse, before the first of them runs)
        self.delta._go(batch, flags | DMH_F_CHECK)
        self.norm._go(flags | DMH_F_CHECK)
        self.conv._go(batch, flags)
        self.delta._go(batch, flags)
        self.norm._go(flags)
        return out


class PortBlock:
    """forward_port_block (src/layers/port_scheduler.mojo:286-482) on fp32 device
    rows, its token mixer the caller's:
      x_mid = x + mix(rmsnorm(x) * input_gamma)
      y     = x_mid + MoE(rmsnorm(x_mid) * post_gamma)
    with the MoE section of an uploaded 4-bit layer.  The mixer's residual and the
    MoE section's norm are one pass."""

    def __init__(self, blk, layer_idx: int, input_gamma=None, post_gamma=None, eps: float = 1e-6):
        self._blk, self._layer = blk, layer_idx
        self._h = h = self._hidden()
        self._before = GatedNorm(blk, h, post=False, edge=True, edge_gamma=input_gamma, eps=eps)
        self._after = GatedNorm(blk, h, post=False, edge=True, edge_gamma=post_gamma, eps=eps)

    def _hidden(self) -> int:
        """The width of the layer as it is now uploaded."""
        dims = self._blk.dims.get(self._layer)
        if dims is None:
            raise _bad(f"layer {self._layer} is not an uploaded 4-bit layer")
        return dims[0]

    def _mixed(self, out, rows):
        """The mixer's output in the block's shape."""
        shape = getattr(out, "shape", ())
        if not shape or shape[-1] != self._h or math.prod(shape) != math.prod(rows):
            raise _bad(f"mix must return {rows[0]} rows of {self._h}")
        return out.reshape(rows)

    def __call__(self, x, mix, xn, x_mid, y):
        """x, xn, x_mid, y [rows][hidden] fp32 device tensors (xn and x_mid are
        overwritten); mix(xn) -> the mixer's output rows [rows][hidden], in fp32,
        fp16 or bf16.  The call takes its place in torch's current stream, as mix
        does: where the block's is another one, each waits for the other."""
        for a, what in ((x, "x"), (xn, "xn"), (x_mid, "x_mid"), (y, "y")):
            if isinstance(a, np.ndarray) or _type(a) != F32 or a.shape != (x.shape[0], self._h) \
                    or not a.is_contiguous() or a.get_device() != self._blk.device:
                raise _bad(f"{what} must be contiguous float32 rows of {self._h} on"
                           f" cuda:{self._blk.device}")
        if self._hidden() != self._h:
            raise _bad(f"layer {self._layer} was replaced by one of {self._hidden()} elements a row")
        rows = (x.shape[0], 1, self._h)
        ours = theirs = None
        if x.is_cuda:
            import torch
            theirs = torch.cuda.current_stream(x.device)
            ours = torch.cuda.ExternalStream(self._blk.stream(), device=x.device)
            if ours.cuda_stream == theirs.cuda_stream:
                ours = None
        if ours is not None:
            ours.wait_stream(theirs)
        try:
            self._before(x.view(rows), y=xn.view(rows))
            if ours is not None:
                theirs.wait_stream(ours)
            try:
                # (a copy where the rows are no view, on the stream that made them)
                out = self._mixed(mix(xn), rows)
            finally:
                if ours is not None:
                    ours.wait_stream(theirs)
            self._after(out, x_mid.view(rows), xn.view(rows), residual=x.view(rows))
            self._blk.forward_device(self._layer, xn.data_ptr(), x.shape[0], y.data_ptr(),
                                     residual_ptr=x_mid.data_ptr())
        finally:
            # (so what `out` was is free only when the block has read it: a tensor must
            # not be recorded on a block's own stream, which may end before the tensor)
            if ours is not None:
                theirs.wait_stream(ours)
        return y
