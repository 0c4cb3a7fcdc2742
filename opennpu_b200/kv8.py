"""An 8-bit KV cache in HBM (onpu_kv8_*): rows of K and V quantised as they are appended, attention over
them, and rows read back. int8 codes, one fp32 scale per (sequence, kv head, block of rows), K and V
apart. Where each sequence stands (``pos``, ``cnt``) is read on the device, so a captured decode step can
be replayed while the sequences grow. The fp32 / bf16 form for one sequence is ``attn.attn_step``."""
import ctypes as C

import torch

from . import libonpu as L


def _need(ok, what):
    if not ok:
        raise L.OnpuError(what)


class KVCache8:
    """B sequences of up to ``rows`` rows, ``heads`` kv heads of ``dim`` (a multiple of 16, at most 256),
    ``block`` (16, 32 or 64) rows to a scale. ``k``, ``v``: int8 [B, heads, rows, dim]; ``k_scale``,
    ``v_scale``: fp32 [B, heads, ceil(rows / block)]. All on the library's device, which has to be the current
    one, in the calls too.

    The calls take, for T tokens of each sequence, ``pos`` (int32 CUDA [B]): the cache row of a
    sequence's first token, and ``cnt`` (int32 CUDA [B], or None for T everywhere): how many of its T
    tokens are real. Token tensors are [B, T, heads, dim] views, bf16 or fp32, with heads dense in a
    token's row and one stride from token to token (a slice of a fused q/k/v projection's rows is one).
    A sequence whose rows are not inside the cache is skipped; ``dense.check_device`` reports it.
    Calls run on the current stream (or ``stream``), asynchronously."""

    def __init__(self, batch, heads, rows, dim, block=32, device="cuda"):
        _need(block in (16, 32, 64), "block: 16, 32 or 64")
        nb = -(-rows // block)
        z = dict(device=device)
        self._bind(torch.zeros(batch, heads, rows, dim, dtype=torch.int8, **z),
                   torch.zeros(batch, heads, rows, dim, dtype=torch.int8, **z),
                   torch.zeros(batch, heads, nb, **z), torch.zeros(batch, heads, nb, **z), block)

    @classmethod
    def from_tensors(cls, k, v, k_scale, v_scale, block=32):
        """A cache over existing tensors (used in place). k and v share their strides, dense along dim;
        so do the scales, dense along the blocks. A slice of sequences of a larger cache is one."""
        self = cls.__new__(cls)
        self._bind(k, v, k_scale, v_scale, block)
        return self

    def _bind(self, k, v, k_scale, v_scale, block):
        _need(k.is_cuda and k.dtype == torch.int8 and k.dim() == 4 and k.stride(3) == 1,
              "k: an int8 CUDA tensor [B, heads, rows, dim], dense along dim")
        _need(v.dtype == torch.int8 and v.shape == k.shape and v.stride() == k.stride() and v.device == k.device,
              "v: like k, with the same strides")
        B, H, S, D = k.shape
        _need(block in (16, 32, 64), "block: 16, 32 or 64")
        # the library runs on the device that is current here (onpu_kv8_attn_ws below checks that it is its own)
        _need(k.get_device() == torch.cuda.current_device(), "k: on the current device")
        nb = -(-S // block)
        for t in (k_scale, v_scale):
            _need(t.dtype == torch.float32 and t.shape == (B, H, nb) and t.device == k.device and
                  t.stride() == k_scale.stride() and (t.stride(2) == 1 or nb == 1),
                  "scales: fp32 [B, heads, ceil(rows / block)] beside k, dense along the blocks")
        self.k, self.v, self.k_scale, self.v_scale, self.block = k, v, k_scale, v_scale, block
        self.batch, self.heads, self.rows, self.dim, self.device, self._dev = B, H, S, D, k.device, k.get_device()
        step = lambda t, i: t.stride(i) if t.shape[i] > 1 else 0      # a lone entry's stride says nothing
        self._desc = L.Kv8Cache(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), B, H, S, D,
                                step(k, 0), step(k, 1), step(k, 2) or D, step(k_scale, 0), step(k_scale, 1), block)
        self._ref = C.addressof(self._desc)
        self._lib = L.require_device()
        L.check(self._lib.onpu_kv8_attn_ws(self._ref, H, 1, 0), "KVCache8")     # sizes, strides, alignment, device
        self._ws = {}                     # (Hq, T, bf16) -> workspace bytes of attn

    # ---------------------------------------------------------------- arguments
    # One condition a tensor: these run before every launch of a decode step.
    def _places(self, pos, cnt):
        shape, dev = (self.batch,), self._dev
        for t in (pos, cnt):
            if t is None and t is not pos:
                return pos.data_ptr(), None
            if t is None or t.dtype is not torch.int32 or t.shape != shape or t.get_device() != dev or \
                    not t.is_contiguous():
                raise L.OnpuError("pos, cnt: int32 [B] on the cache's device, dense")
        return pos.data_ptr(), cnt.data_ptr()

    def _tokens(self, t, heads, name):
        """The token stride of a [B, T, heads, dim] view."""
        try:
            B, T, H, D = t.shape
            sb, st, sh, sd = t.stride()
        except ValueError:
            raise L.OnpuError(f"{name}: [B, T, heads, dim]") from None
        if B != self.batch or D != self.dim or (H != heads and heads) or t.get_device() != self._dev or \
                (t.dtype is not torch.bfloat16 and t.dtype is not torch.float32):
            raise L.OnpuError(f"{name}: bf16 or fp32 [B, T, heads, dim] on the cache's device")
        if sd != 1 or (sh != D and H > 1) or (B > 1 and T > 1 and sb != st * T):
            raise L.OnpuError(f"{name}: heads dense in a token's row, one stride from token to token")
        return st if T > 1 else sb

    def _pair(self, k, v, names):
        ldk, ldv = self._tokens(k, self.heads, names[0]), self._tokens(v, self.heads, names[1])
        if k.shape != v.shape or k.dtype is not v.dtype:
            raise L.OnpuError(f"{names[0]}, {names[1]}: the same tokens and type")
        return ldk, ldv

    def _stream(self, stream):
        # torch.cuda.current_stream(device).cuda_stream, at a twentieth of its host time (2 us)
        return torch._C._cuda_getCurrentRawStream(self._dev) if stream is None else stream.cuda_stream

    # ---------------------------------------------------------------- calls
    def append(self, k, v, pos, cnt=None, stream=None):
        """Quantise the rows k, v [B, T, heads, dim] into cache rows pos .. pos + cnt - 1. A block whose
        scale grows has its older rows re-rounded; a block's first row starts it anew, so rows that were
        appended and then dropped (rejected drafts) are simply written over."""
        p, n = self._places(pos, cnt)
        ldk, ldv = self._pair(k, v, ("k", "v"))
        rc = self._lib.onpu_kv8_append_dev(self._ref, k.data_ptr(), ldk, v.data_ptr(), ldv, k.shape[1],
                                           k.dtype is torch.bfloat16, p, n, self._stream(stream))
        if rc < 0:
            L.check(rc, "onpu_kv8_append_dev")

    def read(self, pos, cnt=None, tokens=None, dtype=torch.bfloat16, out=None, stream=None):
        """Rows pos .. pos + cnt - 1 of every sequence as (k, v), [B, tokens, heads, dim] of ``dtype``; or
        into ``out``, a pair of such tensors. Rows at and past cnt are left as they were (undefined in new
        tensors)."""
        if out is None:
            _need(tokens is not None, "tokens: how many rows of each sequence, where there is no out")
            with torch.cuda.stream(stream):
                out = [torch.empty(self.batch, tokens, self.heads, self.dim, dtype=dtype, device=self.device)
                       for _ in range(2)]
        k, v = out
        p, n = self._places(pos, cnt)
        ldk, ldv = self._pair(k, v, ("out[0]", "out[1]"))
        rc = self._lib.onpu_kv8_read_dev(self._ref, k.data_ptr(), ldk, v.data_ptr(), ldv, k.shape[1],
                                         k.dtype is torch.bfloat16, p, n, self._stream(stream))
        if rc < 0:
            L.check(rc, "onpu_kv8_read_dev")
        return k, v

    def attn(self, q, pos, cnt=None, mask=None, sinks=None, scale=None, out=None, stream=None):
        """Causal attention of q [B, T, Hq, dim] (bf16 or fp32; Hq a multiple of heads, at most 16 times)
        over the cache: token i of a sequence stands at row pos + i, appended before, and sees rows 0 ..
        pos + i. mask: fp32 [B or 1, T or 1, rows], additive, dense along the rows; sinks: fp32 [Hq];
        scale defaults to dim ** -0.5. Returns [B, T, Hq, dim] of q's type; a token whose mask leaves no
        row gets zeros, tokens at and past cnt are left as they were (undefined in a new tensor)."""
        p, n = self._places(pos, cnt)
        ldq = self._tokens(q, None, "q")
        B, T, Hq, D = q.shape
        dev, bf16 = self._dev, q.dtype is torch.bfloat16
        mp, mbs, mts, sp = None, 0, 0, None
        if mask is not None:
            if mask.dtype is not torch.float32 or mask.dim() != 3 or mask.shape[0] not in (1, B) or \
                    mask.shape[1] not in (1, T) or mask.shape[2] != self.rows or mask.get_device() != dev or \
                    (mask.stride(2) != 1 and self.rows > 1):
                raise L.OnpuError("mask: fp32 [B or 1, T or 1, rows] on the cache's device, dense along the rows")
            mp = mask.data_ptr()
            mbs = mask.stride(0) if mask.shape[0] > 1 else 0
            mts = mask.stride(1) if mask.shape[1] > 1 else 0
        if sinks is not None:
            if sinks.dtype is not torch.float32 or sinks.shape != (Hq,) or sinks.get_device() != dev or \
                    not sinks.is_contiguous():
                raise L.OnpuError("sinks: fp32 [Hq] on the cache's device, dense")
            sp = sinks.data_ptr()
        size = self._ws.get((Hq, T, bf16))
        if size is None:
            size = L.check(self._lib.onpu_kv8_attn_ws(self._ref, Hq, T, bf16), "onpu_kv8_attn_ws")
            self._ws[Hq, T, bf16] = size
        if stream is None:
            ws = self.k.new_empty(size)
            out = q.new_empty(q.shape) if out is None else out
        else:
            with torch.cuda.stream(stream):        # memory that this stream may use again
                ws = self.k.new_empty(size)
                out = q.new_empty(q.shape) if out is None else out
        ldo = self._tokens(out, Hq, "out")
        if out.shape[1] != T or out.dtype is not q.dtype:
            raise L.OnpuError("out: q's tokens and type")
        rc = self._lib.onpu_kv8_attn_dev(self._ref, q.data_ptr(), ldq, Hq, T, bf16, p, n, mp, mbs, mts, sp,
                                         D ** -0.5 if scale is None else scale, out.data_ptr(), ldo, ws.data_ptr(),
                                         self._stream(stream))
        if rc < 0:
            L.check(rc, "onpu_kv8_attn_dev")
        return out
