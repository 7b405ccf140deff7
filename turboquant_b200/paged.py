"""Paged cache for requests of different lengths: block tables and slot maps from lengths, norms and rotation of queries
and keys, rows packed into pages and read back, attention of one new token of each request over its pages.

The reference's caches hold one sequence each; its rows (src/cache/storage.rs) are kept here in pages of a fixed number
of tokens, bit for bit as `block_quantize` packs them.  All arithmetic runs in the CUDA library; calls are ordered on the
current stream of the tensors' device.
"""
import ctypes
from dataclasses import dataclass

import torch

from ._lib import TqbPagedAttentionParams, TqbPagedLayer, TqbRopeParams, lib
from .api import ALL_BLOCKS, TQB_ERR_UNSUPPORTED, DecodeOutput, DimensionMismatch, QuantNormMode, TqbRuntimeError, check

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TICKET_BYTES = 16384   # TQB_PAGED_TICKET_BYTES
_INTERLEAVED, _NO_NORM, _POSITIONS_64 = 1, 2, 4
_PLAN_STATUS = {1: "not enough free pages", 2: "a request's length is negative or beyond its block table",
                3: "more new tokens than the plan's capacity"}


def _code(dt):
    code = _DTYPES.get(dt)
    if code is None:
        raise TypeError(f"unsupported dtype {dt}")
    return code


def _call(device, fn, *args):
    """fn(*args, stream) with the tensors' device current."""
    index = device.index
    if index == torch.cuda.current_device():
        check(fn(*args, torch.cuda.current_stream(index).cuda_stream))
    else:
        with torch.cuda.device(index):
            check(fn(*args, torch.cuda.current_stream(index).cuda_stream))


def _want(name, t, dtype, shape, device):
    """A dense tensor of this dtype and shape (None: any extent) on `device`."""
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.dim() != len(shape) or any(s is not None and s != n for s, n in zip(shape, t.shape)):
        raise DimensionMismatch(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")


def _cuda(name, t):
    if not t.is_cuda:
        raise ValueError(f"{name}: expected a CUDA tensor")
    return t.device


def _rows(name, t, heads, dim, device):
    """A tensor [tokens, heads, dim] whose rows the kernels can read where they lie, else a dense copy of it."""
    if t.dim() != 3 or t.shape[2] != dim or (heads is not None and t.shape[1] != heads):
        raise DimensionMismatch(f"{name}: expected shape (tokens, {heads or 'heads'}, {dim}), got {tuple(t.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got {t.device}")
    s0, s1, s2 = t.stride()
    e = 16 // t.element_size()
    if s2 != 1 or s0 % e or s1 % e or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _out_rows(name, t, like, device):
    if t.dtype != like.dtype or t.shape != like.shape:
        raise DimensionMismatch(f"{name}: expected {like.dtype} of shape {tuple(like.shape)}")
    if t.device != device:
        raise ValueError(f"{name}: expected a tensor on {device}, got {t.device}")
    s0, s1, s2 = t.stride()
    e, (n, h, d) = 16 // t.element_size(), t.shape
    if s2 != 1 or s0 % e or s1 % e or t.data_ptr() % 16 or (h > 1 and s1 < d) or (n > 1 and s0 < (h - 1) * s1 + d):
        raise ValueError(f"{name}: rows must be dense, 16-byte aligned and apart from one another")


# ---------------------------------------------------------------------------------------
# Block tables and slot maps
# ---------------------------------------------------------------------------------------
@dataclass
class PagedStep:
    """One step of a batch: where its new tokens go.  slots, positions [capacity] (behind the last token -1 and 0),
    cu [requests + 1], kv_lens [requests] with the new tokens counted, state: {free pages, 0, status, 0}."""
    slots: torch.Tensor
    positions: torch.Tensor
    cu: torch.Tensor
    kv_lens: torch.Tensor
    state: torch.Tensor

    def check(self):
        """Raises if the step could not be planned; waits for the device."""
        status = int(self.state[2])
        if status:
            err = TqbRuntimeError(_PLAN_STATUS.get(status, f"plan status {status}"))
            err.status = status
            raise err


def _plan_shapes(seq_lens, block_table, free_pages, state):
    dev = _cuda("seq_lens", seq_lens)
    n = seq_lens.shape[0] if seq_lens.dim() == 1 else -1
    _want("seq_lens", seq_lens, torch.int32, (None,), dev)
    _want("block_table", block_table, torch.int32, (n, None), dev)
    _want("free_pages", free_pages, torch.int32, (None,), dev)
    _want("state", state, torch.int32, (4,), dev)
    return dev, n


def paged_plan(seq_lens, new_tokens, block_table, free_pages, state, page_size, capacity, kv_lens=None, state_out=None):
    """Block tables, slot map and positions of a step from the requests' lengths (tqb_paged_plan).

    seq_lens, new_tokens [requests], block_table [requests, blocks] (new entries are written in place), free_pages and
    state int32; the first state[0] entries of free_pages are the free pages.  kv_lens and state_out are made new unless
    given; they may be seq_lens and state themselves.  Returns a PagedStep; `check()` on it says whether the step fitted."""
    dev, n = _plan_shapes(seq_lens, block_table, free_pages, state)
    _want("new_tokens", new_tokens, torch.int32, (n,), dev)
    if capacity < 0:
        raise ValueError("capacity must not be negative")
    slots = torch.empty(capacity, dtype=torch.int64, device=dev)
    positions = torch.empty(capacity, dtype=torch.int32, device=dev)
    cu = torch.empty(n + 1, dtype=torch.int32, device=dev)
    if kv_lens is None:
        kv_lens = torch.empty(n, dtype=torch.int32, device=dev)
    else:
        _want("kv_lens", kv_lens, torch.int32, (n,), dev)
    if state_out is None:
        state_out = torch.empty(4, dtype=torch.int32, device=dev)
    else:
        _want("state_out", state_out, torch.int32, (4,), dev)
    blocks = block_table.shape[1]
    _call(dev, lib.tqb_paged_plan, seq_lens.data_ptr(), new_tokens.data_ptr(), n, block_table.data_ptr(), blocks, blocks,
          free_pages.data_ptr(), state.data_ptr(), page_size, slots.data_ptr(), positions.data_ptr(), capacity, cu.data_ptr(),
          kv_lens.data_ptr(), state_out.data_ptr())
    return PagedStep(slots, positions, cu, kv_lens, state_out)


def paged_release(mask, seq_lens, block_table, free_pages, state, page_size):
    """Gives the pages of the requests with mask[r] back to free_pages (tqb_paged_release): in place."""
    dev, n = _plan_shapes(seq_lens, block_table, free_pages, state)
    if mask.dtype == torch.bool:
        mask = mask.view(torch.uint8)
    _want("mask", mask, torch.uint8, (n,), dev)
    blocks = block_table.shape[1]
    _call(dev, lib.tqb_paged_release, mask.data_ptr(), seq_lens.data_ptr(), n, block_table.data_ptr(), blocks, blocks,
          free_pages.data_ptr(), free_pages.shape[0], state.data_ptr(), page_size)


# ---------------------------------------------------------------------------------------
# Norms of queries and keys with the position rotation
# ---------------------------------------------------------------------------------------
class QkNormRope:
    """RMS norm of each head of queries and keys and the position rotation, in one pass (tqb_qk_norm_rope).

    inv_freq [rot_dim / 2] f32 (an empty tensor: no rotation); q_weight, k_weight [head_dim] of the queries' dtype, or None
    for ones; norm=False leaves the norms out; interleaved rotates neighbouring elements together instead of halves."""

    def __init__(self, inv_freq, q_weight=None, k_weight=None, eps=1e-6, norm=True, interleaved=False):
        self.device = _cuda("inv_freq", inv_freq)
        _want("inv_freq", inv_freq, torch.float32, (None,), self.device)
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None:
                _want(name, w, w.dtype, (None,), self.device)
                _code(w.dtype)
                if w.data_ptr() % 16:
                    raise ValueError(f"{name}: expected a 16-byte aligned tensor")
        self.inv_freq, self.q_weight, self.k_weight = inv_freq, q_weight, k_weight
        self.eps, self.norm, self.interleaved = float(eps), bool(norm), bool(interleaved)

    def _params(self, q, k, positions):
        """The argument block for q, k (either may be None) without outputs."""
        x = q if q is not None else k
        n, d, dt = x.shape[0], x.shape[2], x.dtype
        p = TqbRopeParams()
        p.dtype, p.num_tokens, p.head_dim, p.eps = _code(dt), n, d, self.eps
        p.rot_dim = 2 * self.inv_freq.shape[0]
        flags = (_INTERLEAVED if self.interleaved else 0) | (0 if self.norm else _NO_NORM)
        if p.rot_dim:
            if positions.dtype == torch.int64:
                flags |= _POSITIONS_64
            elif positions.dtype != torch.int32:
                raise TypeError(f"positions: expected int32 or int64, got {positions.dtype}")
            _want("positions", positions, positions.dtype, (n,), self.device)
            p.positions, p.inv_freq = positions.data_ptr(), self.inv_freq.data_ptr()
        p.flags = flags
        for w, name in ((self.q_weight, "q_weight"), (self.k_weight, "k_weight")):
            if w is not None and self.norm:
                if w.dtype != dt or w.shape[0] != d:
                    raise DimensionMismatch(f"{name}: expected {dt} of length {d}, got {w.dtype} of length {w.shape[0]}")
                setattr(p, name, w.data_ptr())
        if q is not None:
            p.q, p.num_q_heads = q.data_ptr(), q.shape[1]
            p.q_token_stride, p.q_head_stride, _ = q.stride()
        if k is not None:
            if k.dtype != dt or k.shape[0] != n:
                raise DimensionMismatch(f"k: expected {dt} with {n} tokens, got {k.dtype} with {k.shape[0]}")
            p.k, p.num_kv_heads = k.data_ptr(), k.shape[1]
            p.k_token_stride, p.k_head_stride, _ = k.stride()
        return p

    def __call__(self, q, k, positions, q_out=None, k_out=None):
        """q [tokens, query heads, dim], k [tokens, KV heads, dim] -> (q_out, k_out); the outputs may be q and k themselves."""
        d = q.shape[-1]
        qi, ki = _rows("q", q, None, d, self.device), _rows("k", k, None, d, self.device)
        p = self._params(qi, ki, positions)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        else:
            _out_rows("q_out", q_out, q, self.device)
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=self.device)
        else:
            _out_rows("k_out", k_out, k, self.device)
        p.q_out, p.k_out = q_out.data_ptr(), k_out.data_ptr()
        p.q_out_token_stride, p.q_out_head_stride, _ = q_out.stride()
        p.k_out_token_stride, p.k_out_head_stride, _ = k_out.stride()
        _call(self.device, lib.tqb_qk_norm_rope, ctypes.byref(p))
        return q_out, k_out


# ---------------------------------------------------------------------------------------
# The pages of one layer
# ---------------------------------------------------------------------------------------
class PagedLayer:
    """The pages of one layer: k_indices, v_indices [pages, KV heads, page_size, head_dim * bits / 8] u8 and k_scales,
    v_scales [pages, KV heads, page_size, head_dim / 32] int16 (f16 bits).  The tensors stay the caller's."""

    def __init__(self, k_indices, k_scales, v_indices, v_scales, bits):
        dev = _cuda("k_indices", k_indices)
        if k_indices.dim() != 4 or k_scales.dim() != 4:
            raise DimensionMismatch("expected arrays [pages, KV heads, page_size, ...]")
        pages, heads, page, _ = k_indices.shape
        dim = 32 * k_scales.shape[3]
        for name, t in (("k_indices", k_indices), ("v_indices", v_indices)):
            _want(name, t, torch.uint8, (pages, heads, page, dim * bits // 8), dev)
        for name, t in (("k_scales", k_scales), ("v_scales", v_scales)):
            _want(name, t, torch.int16, (pages, heads, page, dim // 32), dev)
        self.tensors = (k_indices, k_scales, v_indices, v_scales)
        self.device, self.bits, self.head_dim = dev, bits, dim
        self.num_pages, self.num_kv_heads, self.page_size = pages, heads, page
        self._c = TqbPagedLayer(k_indices.data_ptr(), k_scales.data_ptr(), v_indices.data_ptr(), v_scales.data_ptr(), pages, heads, page,
                                dim, bits, 0)
        self._ref = ctypes.byref(self._c)
        check(lib.tqb_paged_dequantize(self._ref, None, 0, None, None, 0, None))   # checks the description, launches nothing

    def _slots(self, slots, n):
        _want("slots", slots, torch.int64, (n,), self.device)
        return slots.data_ptr()

    def append(self, k, v, slots):
        """Packs k, v [tokens, KV heads, dim] into their slots; a slot of -1 leaves a token out."""
        k = _rows("k", k, self.num_kv_heads, self.head_dim, self.device)
        v = _rows("v", v, self.num_kv_heads, self.head_dim, self.device)
        if v.dtype != k.dtype or v.shape != k.shape:
            raise DimensionMismatch("k and v differ in dtype or shape")
        n = k.shape[0]
        sk, sv = k.stride(), v.stride()
        _call(self.device, lib.tqb_paged_append, self._ref, k.data_ptr(), sk[0], sk[1], v.data_ptr(), sv[0], sv[1], _code(k.dtype),
              self._slots(slots, n), n)

    def append_rope(self, rope, q, k, v, positions, slots, q_out=None):
        """Norms and rotation of q and k (`rope`: a QkNormRope), the keys and v packed into their slots, in one launch.
        Returns the rotated queries."""
        q = _rows("q", q, None, self.head_dim, self.device)
        k = _rows("k", k, self.num_kv_heads, self.head_dim, self.device)
        v = _rows("v", v, self.num_kv_heads, self.head_dim, self.device)
        if v.dtype != k.dtype or v.shape != k.shape:
            raise DimensionMismatch("k and v differ in dtype or shape")
        if rope.device != self.device:
            raise ValueError(f"rope: expected tensors on {self.device}, got {rope.device}")
        p = rope._params(q, k, positions)
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        else:
            _out_rows("q_out", q_out, q, self.device)
        p.q_out = q_out.data_ptr()
        p.q_out_token_stride, p.q_out_head_stride, _ = q_out.stride()
        sv = v.stride()
        _call(self.device, lib.tqb_paged_append_rope, self._ref, ctypes.byref(p), v.data_ptr(), sv[0], sv[1],
              self._slots(slots, k.shape[0]))
        return q_out

    def dequantize(self, slots, dtype=torch.float32):
        """The rows at `slots`: (k, v) [n, KV heads, dim]; rows of zeros where a slot lies outside the pages."""
        n = slots.shape[0]
        k = torch.empty((n, self.num_kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        _call(self.device, lib.tqb_paged_dequantize, self._ref, self._slots(slots, n), n, k.data_ptr(), v.data_ptr(), _code(dtype))
        return k, v

    def attend_scratch(self, num_q_heads):
        """A work area for `attend`, its tickets zero-filled once.  Two calls that may run at the same time need one each."""
        n = int(lib.tqb_paged_scratch_bytes(num_q_heads, self.num_kv_heads, self.head_dim))
        scratch = torch.empty(n, dtype=torch.uint8, device=self.device)
        scratch[:_TICKET_BYTES].zero_()
        return scratch

    def attend(self, q, block_table, kv_lens, softmax_scale, out=None, scratch=None):
        """Attention of one new token of each request over its pages: q [requests, query heads, dim] -> the same shape.
        block_table [requests, blocks] and kv_lens [requests] int32; a request without tokens gets zeros."""
        n, hq, d = q.shape
        q = _rows("q", q, None, self.head_dim, self.device)
        if q.stride(1) != d or (n > 1 and q.stride(0) < hq * d):
            q = q.contiguous()
        _want("block_table", block_table, torch.int32, (n, None), self.device)
        _want("kv_lens", kv_lens, torch.int32, (n,), self.device)
        if out is None:
            out = torch.empty((n, hq, d), dtype=q.dtype, device=self.device)
        else:
            _want("out", out, out.dtype, (n, hq, d), self.device)
        if scratch is None:
            scratch = self.attend_scratch(hq)
        else:
            _want("scratch", scratch, torch.uint8, (None,), self.device)
        blocks = block_table.shape[1]
        p = TqbPagedAttentionParams(q.data_ptr(), out.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), scratch.data_ptr(),
                                    scratch.shape[0], q.stride(0) if n > 1 else 0, blocks, blocks, n, hq, _code(q.dtype),
                                    _code(out.dtype), softmax_scale)
        _call(self.device, lib.tqb_paged_attention, self._ref, ctypes.byref(p))
        return out


class PagedPqoCache:
    """A paged cache of all layers: pages, block tables, lengths and the list of free pages of up to `max_requests` running
    requests.  The counterpart of PqoCache (src/cache/pqo.rs:21-236) for requests of different lengths.

        step = cache.plan(new_tokens, capacity)                # once a step
        q = cache.append_rope(layer, rope, q, k, v, step)      # each layer
        out = cache.decode(layer, q, step, att).fused          # steps of one token a request
    """

    def __init__(self, config, num_pages, page_size=64, max_requests=64, max_blocks=None, device=None):
        if config.norm_mode != QuantNormMode.MaxNorm or config.outlier_blocks not in (ALL_BLOCKS, config.num_blocks()):
            check(TQB_ERR_UNSUPPORTED)
        if config.batch != 1:
            raise DimensionMismatch("a paged cache takes its requests from the block table: batch must be 1")
        self.config, self.page_size = config, page_size
        dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
        rows = (num_pages, config.num_kv_heads, page_size)

        def arrays():
            return (torch.zeros((*rows, config.packed_dim()), dtype=torch.uint8, device=dev),
                    torch.zeros((*rows, config.num_blocks()), dtype=torch.int16, device=dev))

        self.layers = [PagedLayer(*arrays(), *arrays(), config.bits) for _ in range(config.num_layers)]
        self.device = self.layers[0].device if self.layers else dev
        blocks = num_pages if max_blocks is None else max_blocks
        self.block_table = torch.full((max_requests, blocks), -1, dtype=torch.int32, device=dev)
        self.seq_lens = torch.zeros(max_requests, dtype=torch.int32, device=dev)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, dtype=torch.int32, device=dev)
        self.state = torch.tensor([num_pages, 0, 0, 0], dtype=torch.int32, device=dev)
        self._scratch = {}

    def plan(self, new_tokens, capacity):
        """Pages, slots and positions for new_tokens [max_requests] int32 of each request; `step.check()` tells whether
        they fitted.  The step's kv_lens and state are the cache's own and go on with its next plan."""
        return paged_plan(self.seq_lens, new_tokens, self.block_table, self.free_pages, self.state, self.page_size, capacity,
                          kv_lens=self.seq_lens, state_out=self.state)

    def release(self, mask):
        """Ends the requests with mask[r] (bool or u8 [max_requests]); their rows may be used by new ones."""
        paged_release(mask, self.seq_lens, self.block_table, self.free_pages, self.state, self.page_size)

    def append(self, layer, k, v, step):
        self._layer(layer).append(k, v, step.slots[: k.shape[0]])

    def append_rope(self, layer, rope, q, k, v, step, q_out=None):
        n = k.shape[0]
        return self._layer(layer).append_rope(rope, q, k, v, step.positions[:n], step.slots[:n], q_out=q_out)

    def dequantize(self, layer, slots, dtype=torch.float32):
        return self._layer(layer).dequantize(slots, dtype)

    def decode(self, layer, q, step, config, out=None, scratch=None):
        """Attention of q [max_requests, query heads, dim] over everything stored: DecodeOutput with `fused` set.
        Without `scratch` the cache keeps one for each stream, and a call that is being captured gets its own."""
        at = self._layer(layer)
        if scratch is None and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self.device).cuda_stream
            scratch = self._scratch.get(stream)
            if scratch is None:
                scratch = self._scratch[stream] = at.attend_scratch(q.shape[1])
        return DecodeOutput(fused=at.attend(q, self.block_table, step.kv_lens, config.softmax_scale, out=out, scratch=scratch))

    def _layer(self, layer):
        if not 0 <= layer < len(self.layers):
            check(4)
        return self.layers[layer]

    def memory_usage(self):
        return sum(t.numel() * t.element_size() for x in self.layers for t in x.tensors)
