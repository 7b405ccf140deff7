"""Paged cache for requests of different lengths: block tables and slot maps from lengths, norms and rotation of queries
and keys, rows packed into pages and read back, attention of one new token of each request over its pages.

The reference's caches hold one sequence each; its rows (src/cache/storage.rs) are kept here in pages of a fixed number
of tokens, bit for bit as `block_quantize` packs them.  All arithmetic runs in the CUDA library; calls are ordered on the
current stream of the tensors' device.
"""
import struct
from dataclasses import dataclass

import torch

from ._lib import lib
from .api import ALL_BLOCKS, TQB_ERR_UNSUPPORTED, DecodeOutput, DimensionMismatch, QuantNormMode, TqbRuntimeError, check

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_TICKET_BYTES = 16384   # TQB_PAGED_TICKET_BYTES
_INTERLEAVED, _NO_NORM, _POSITIONS_64 = 1, 2, 4
_PLAN_STATUS = {1: "not enough free pages", 2: "a request's length is negative or beyond its block table",
                3: "more new tokens than the plan's capacity"}
# The C structures (tqb200.h), packed in one go for each call: these calls are short, and so is their way to the launch.
_LAYER = struct.Struct("@4P6i")                 # tqb_paged_layer
_ROPE = struct.Struct("@4P8q4P7if")             # tqb_rope_params
_ATTEND = struct.Struct("@5PN2q5if")            # tqb_paged_attention_params

_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _code(dt):
    code = _DTYPES.get(dt)
    if code is None:
        raise TypeError(f"unsupported dtype {dt}")
    return code


def _call(index, fn, *args):
    """fn(*args, stream) with the tensors' device current."""
    if index == _current_device():
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        check(status)


def _eager_stream(index):
    """The handle of the device's current stream, or None while it is being captured."""
    if index != _current_device():
        with torch.cuda.device(index):
            return _eager_stream(index)
    return None if torch.cuda.is_current_stream_capturing() else _raw_stream(index)


def _device(name, t):
    index = t.get_device()
    if index < 0:
        raise ValueError(f"{name}: expected a CUDA tensor")
    return index


def _want(name, t, dtype, shape, index):
    """The address of a dense tensor of this dtype and shape on the device."""
    if t.dtype is not dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise DimensionMismatch(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name}: expected a tensor on cuda:{index}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{name}: expected a contiguous tensor")
    return t.data_ptr()


def _rows(name, t, shape, index):
    """(tensor, address, token stride, head stride) of rows [tokens, heads, dim]: where they lie if the kernels can read them
    there, else of a dense copy."""
    if t.shape != shape:
        raise DimensionMismatch(f"{name}: expected shape {tuple(shape)}, got {tuple(t.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name}: expected a tensor on cuda:{index}, got {t.device}")
    at, (s0, s1, s2), e = t.data_ptr(), t.stride(), 16 // t.element_size()
    if s2 != 1 or s0 % e or s1 % e or at % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        at, (s0, s1, s2) = t.data_ptr(), t.stride()
    return t, at, s0, s1


def _out_rows(name, t, like, index):
    """(address, token stride, head stride) of rows to be written."""
    if t.dtype is not like.dtype or t.shape != like.shape:
        raise DimensionMismatch(f"{name}: expected {like.dtype} of shape {tuple(like.shape)}")
    if t.get_device() != index:
        raise ValueError(f"{name}: expected a tensor on cuda:{index}, got {t.device}")
    at, (s0, s1, s2), e, (n, h, d) = t.data_ptr(), t.stride(), 16 // t.element_size(), t.shape
    by_token, by_head = n < 2 or s0 >= (h - 1) * s1 + d, h < 2 or s1 >= (n - 1) * s0 + d   # the rows of a token, of a head lie together
    if s2 != 1 or s0 % e or s1 % e or at % 16 or (h > 1 and s1 < d) or (n > 1 and s0 < d) or not (by_token or by_head):
        raise ValueError(f"{name}: rows must be dense, 16-byte aligned and apart from one another")
    return at, s0, s1


def _empty_like(like, n, heads, dim):
    """A dense tensor of like's type and this shape, which is like's (empty_like is the shorter way, 1.4 us against 1.9)."""
    return torch.empty_like(like) if like.is_contiguous() else like.new_empty((n, heads, dim))


def _made(out, name, like, n, heads, dim, index):
    """(tensor, its rows as _out_rows gives them) of an output, made here unless given."""
    if out is not None:
        return out, _out_rows(name, out, like, index)
    out = _empty_like(like, n, heads, dim)
    return out, (out.data_ptr(), heads * dim, dim)


def _three(name, t):
    if t.dim() != 3:
        raise DimensionMismatch(f"{name}: expected [tokens, heads, dim], got {tuple(t.shape)}")
    return t.shape


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
        _check_plan(int(self.state[2]))


def _check_plan(status):
    if status:
        err = TqbRuntimeError(_PLAN_STATUS.get(status, f"plan status {status}"))
        err.status = status
        raise err


def _plan_args(seq_lens, block_table, free_pages, state):
    index = _device("seq_lens", seq_lens)
    if seq_lens.dim() != 1 or block_table.dim() != 2 or free_pages.dim() != 1:
        raise DimensionMismatch("expected seq_lens [requests], block_table [requests, blocks] and free_pages [pages]")
    n, blocks = seq_lens.shape[0], block_table.shape[1]
    i32 = torch.int32
    return (index, n, blocks, _want("seq_lens", seq_lens, i32, (n,), index), _want("block_table", block_table, i32, (n, blocks), index),
            _want("free_pages", free_pages, i32, free_pages.shape, index), _want("state", state, i32, (4,), index))


def paged_plan(seq_lens, new_tokens, block_table, free_pages, state, page_size, capacity, kv_lens=None, state_out=None, failed=None):
    """Block tables, slot map and positions of a step from the requests' lengths (tqb_paged_plan_bounded).

    seq_lens, new_tokens [requests], block_table [requests, blocks] (new entries are written in place), free_pages and
    state int32; the first state[0] entries of free_pages are the free pages.  kv_lens and state_out are made new unless
    given; they may be seq_lens and state themselves.  Returns a PagedStep; `check()` on it says whether the step fitted (with
    state[0] beyond the list's length no page is to be had).  failed [1] int32, if given, gets the status of every plan and
    release that did not fit, and keeps it when later ones do."""
    index, n, blocks, seq, table, free, st = _plan_args(seq_lens, block_table, free_pages, state)
    new = _want("new_tokens", new_tokens, torch.int32, (n,), index)
    if capacity < 0:
        raise ValueError("capacity must not be negative")
    dev = seq_lens.device
    slots = torch.empty(capacity, dtype=torch.int64, device=dev)
    made = torch.empty(capacity + n + 1 + (n if kv_lens is None else 0) + (4 if state_out is None else 0), dtype=torch.int32, device=dev)
    parts = [capacity, n + 1]
    if kv_lens is None:
        parts.append(n)
    else:
        _want("kv_lens", kv_lens, torch.int32, (n,), index)
    if state_out is None:
        parts.append(4)
    else:
        _want("state_out", state_out, torch.int32, (4,), index)
    parts = list(made.split_with_sizes(parts))
    positions, cu = parts[0], parts[1]
    if state_out is None:
        state_out = parts.pop()
    if kv_lens is None:
        kv_lens = parts.pop()
    _call(index, lib.tqb_paged_plan_bounded, seq, new, n, table, blocks, blocks, free, free_pages.shape[0], st, page_size, slots.data_ptr(),
          positions.data_ptr(), capacity, cu.data_ptr(), kv_lens.data_ptr(), state_out.data_ptr(),
          None if failed is None else _want("failed", failed, torch.int32, (1,), index))
    return PagedStep(slots, positions, cu, kv_lens, state_out)


def paged_release(mask, seq_lens, block_table, free_pages, state, page_size):
    """Gives the pages of the requests with mask[r] back to free_pages (tqb_paged_release): in place.  A page that requests
    share goes back once, when the last of them ends."""
    index, n, blocks, seq, table, free, st = _plan_args(seq_lens, block_table, free_pages, state)
    if mask.dtype is torch.bool:
        mask = mask.view(torch.uint8)
    _call(index, lib.tqb_paged_release, _want("mask", mask, torch.uint8, (n,), index), seq, n, table, blocks, blocks, free,
          free_pages.shape[0], st, page_size)


# ---------------------------------------------------------------------------------------
# Norms of queries and keys with the position rotation
# ---------------------------------------------------------------------------------------
class QkNormRope:
    """RMS norm of each head of queries and keys and the position rotation, in one pass (tqb_qk_norm_rope).

    inv_freq [rot_dim / 2] f32 (an empty tensor: no rotation); q_weight, k_weight [head_dim] of the queries' dtype, or None
    for ones; norm=False leaves the norms out; interleaved rotates neighbouring elements together instead of halves."""

    def __init__(self, inv_freq, q_weight=None, k_weight=None, eps=1e-6, norm=True, interleaved=False):
        self.index = _device("inv_freq", inv_freq)
        if inv_freq.dim() != 1:
            raise DimensionMismatch("inv_freq: expected [rot_dim / 2]")
        self._freq = _want("inv_freq", inv_freq, torch.float32, inv_freq.shape, self.index)
        for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
            if w is not None:
                _code(w.dtype)
                if w.dim() != 1 or _want(name, w, w.dtype, w.shape, self.index) % 16:
                    raise ValueError(f"{name}: expected a 16-byte aligned vector")
        self.inv_freq, self.q_weight, self.k_weight = inv_freq, q_weight, k_weight
        self.eps, self.norm, self.interleaved = float(eps), bool(norm), bool(interleaved)
        self._rot = 2 * inv_freq.shape[0]
        self._flags = (_INTERLEAVED if self.interleaved else 0) | (0 if self.norm else _NO_NORM)

    def _weight(self, name, w, dt, d):
        if w is None or not self.norm:
            return None
        if w.dtype is not dt or w.shape[0] != d:
            raise DimensionMismatch(f"{name}: expected {dt} of length {d}, got {w.dtype} of length {w.shape[0]}")
        return w.data_ptr()

    def _params(self, q, q_out, k, k_out, n, hq, hkv, d, dt, positions):
        """The argument block; q .. k_out are (address, token stride, head stride)."""
        flags, at = self._flags, 0
        if self._rot:
            if positions.dtype is torch.int64:
                flags |= _POSITIONS_64
            elif positions.dtype is not torch.int32:
                raise TypeError(f"positions: expected int32 or int64, got {positions.dtype}")
            at = _want("positions", positions, positions.dtype, (n,), self.index)
        wq, wk = self._weight("q_weight", self.q_weight, dt, d), self._weight("k_weight", self.k_weight, dt, d)
        return _ROPE.pack(q[0], q_out[0], k[0], k_out[0], q[1], q[2], q_out[1], q_out[2], k[1], k[2], k_out[1], k_out[2], wq or 0, wk or 0, at,
                          self._freq, n, hq, hkv, d, self._rot, _code(dt), flags, self.eps)

    def __call__(self, q, k, positions, q_out=None, k_out=None):
        """q [tokens, query heads, dim], k [tokens, KV heads, dim] -> (q_out, k_out); the outputs may be q and k themselves."""
        index, dt = self.index, q.dtype
        n, hq, d = _three("q", q)
        hkv = _three("k", k)[1]
        if k.dtype is not dt:
            raise DimensionMismatch(f"k: expected {dt}, got {k.dtype}")
        qi, ki = _rows("q", q, q.shape, index), _rows("k", k, (n, hkv, d), index)
        q_out, qo = _made(q_out, "q_out", q, n, hq, d, index)
        k_out, ko = _made(k_out, "k_out", k, n, hkv, d, index)
        _call(index, lib.tqb_qk_norm_rope, self._params(qi[1:], qo, ki[1:], ko, n, hq, hkv, d, dt, positions))
        return q_out, k_out


# ---------------------------------------------------------------------------------------
# The pages of one layer
# ---------------------------------------------------------------------------------------
class PagedLayer:
    """The pages of one layer: k_indices, v_indices [pages, KV heads, page_size, head_dim * bits / 8] u8 and k_scales,
    v_scales [pages, KV heads, page_size, head_dim / 32] int16 (f16 bits).  The tensors stay the caller's."""

    def __init__(self, k_indices, k_scales, v_indices, v_scales, bits):
        self.index = _device("k_indices", k_indices)
        if k_indices.dim() != 4 or k_scales.dim() != 4:
            raise DimensionMismatch("expected arrays [pages, KV heads, page_size, ...]")
        pages, heads, page, _ = k_indices.shape
        dim = 32 * k_scales.shape[3]
        codes, blocks = (pages, heads, page, dim * bits // 8), (pages, heads, page, dim // 32)
        self._c = _LAYER.pack(_want("k_indices", k_indices, torch.uint8, codes, self.index), _want("k_scales", k_scales, torch.int16, blocks, self.index),
                              _want("v_indices", v_indices, torch.uint8, codes, self.index), _want("v_scales", v_scales, torch.int16, blocks, self.index),
                              pages, heads, page, dim, bits, 0)
        self.tensors = (k_indices, k_scales, v_indices, v_scales)
        self.device, self.bits, self.head_dim = k_indices.device, bits, dim
        self.num_pages, self.num_kv_heads, self.page_size = pages, heads, page
        check(lib.tqb_paged_dequantize(self._c, None, 0, None, None, 0, None))   # checks the description, launches nothing

    def _slots(self, slots, n):
        return _want("slots", slots, torch.int64, (n,), self.index)

    def _kv(self, k, v):
        n = k.shape[0]
        shape = (n, self.num_kv_heads, self.head_dim)
        if v.dtype is not k.dtype:
            raise DimensionMismatch(f"k and v differ in dtype: {k.dtype}, {v.dtype}")
        return n, _rows("k", k, shape, self.index), _rows("v", v, shape, self.index)

    def append(self, k, v, slots):
        """Packs k, v [tokens, KV heads, dim] into their slots; a slot of -1 leaves a token out."""
        n, k, v = self._kv(k, v)
        _call(self.index, lib.tqb_paged_append, self._c, k[1], k[2], k[3], v[1], v[2], v[3], _code(k[0].dtype), self._slots(slots, n), n)

    def append_rope(self, rope, q, k, v, positions, slots, q_out=None):
        """Norms and rotation of q and k (`rope`: a QkNormRope), the keys and v packed into their slots, in one launch.
        Returns the rotated queries."""
        n, k, v = self._kv(k, v)
        hq, d, index = _three("q", q)[1], self.head_dim, self.index
        qi = _rows("q", q, (n, hq, d), index)
        if q.dtype is not k[0].dtype:
            raise DimensionMismatch(f"q and k differ in dtype: {q.dtype}, {k[0].dtype}")
        if rope.index != index:
            raise ValueError(f"rope: expected tensors on cuda:{index}, got cuda:{rope.index}")
        q_out, qo = _made(q_out, "q_out", q, n, hq, d, index)
        p = rope._params(qi[1:], qo, k[1:], (0, 0, 0), n, hq, self.num_kv_heads, d, q.dtype, positions)
        _call(index, lib.tqb_paged_append_rope, self._c, p, v[1], v[2], v[3], self._slots(slots, n))
        return q_out

    def dequantize(self, slots, dtype=torch.float32):
        """The rows at `slots`: (k, v) [n, KV heads, dim]; rows of zeros where a slot lies outside the pages."""
        n = slots.shape[0]
        at = self._slots(slots, n)
        k = slots.new_empty((n, self.num_kv_heads, self.head_dim), dtype=dtype)
        v = torch.empty_like(k)
        _call(self.index, lib.tqb_paged_dequantize, self._c, at, n, k.data_ptr(), v.data_ptr(), _code(dtype))
        return k, v

    def attend_scratch(self, num_q_heads):
        """A work area for `attend`, its tickets zero-filled once.  Two calls that may run at the same time need one each."""
        n = int(lib.tqb_paged_scratch_bytes(num_q_heads, self.num_kv_heads, self.head_dim))
        scratch = torch.empty(n, dtype=torch.uint8, device=self.device)
        scratch[:_TICKET_BYTES].zero_()
        return scratch

    def attend(self, q, block_table, kv_lens, softmax_scale, out=None, scratch=None, cu=None):
        """Attention of one new token of each request over its pages: q [requests, query heads, dim] -> the same shape.
        block_table [requests, blocks] and kv_lens [requests] int32; a request without tokens gets zeros.

        With cu [requests + 1] (a PagedStep's) the rows of q and out are the step's tokens: row cu[r] is that of request r, if
        it brings exactly one token.  Other rows of a given `out` stay as they are; of one made here they are zeros."""
        index, d = self.index, self.head_dim
        n, hq, _ = _three("q", q)
        qi, at, s0, s1 = _rows("q", q, (n, hq, d), index)
        if s1 != d or (n > 1 and s0 < hq * d):   # heads one behind the other
            qi = qi.contiguous() if not qi.is_contiguous() else qi.clone()
            at, s0 = qi.data_ptr(), hq * d
        if block_table.dim() != 2:
            raise DimensionMismatch(f"block_table: expected [requests, blocks], got {tuple(block_table.shape)}")
        requests, blocks = n if cu is None else block_table.shape[0], block_table.shape[1]
        table = _want("block_table", block_table, torch.int32, (requests, blocks), index)
        lens = _want("kv_lens", kv_lens, torch.int32, (requests,), index)
        if out is None:
            out = _empty_like(q, n, hq, d) if cu is None else q.new_zeros((n, hq, d))
            to = out.data_ptr()
        else:
            to = _want("out", out, out.dtype, (n, hq, d), index)
        if scratch is None:
            scratch = self.attend_scratch(hq)
        work = _want("scratch", scratch, torch.uint8, scratch.shape, index)
        p = _ATTEND.pack(at, to, table, lens, work, scratch.numel(), s0 if n > 1 else 0, blocks, blocks, requests, hq, _code(q.dtype), _code(out.dtype), softmax_scale)
        if cu is None:
            _call(index, lib.tqb_paged_attention, self._c, p)
        elif n:
            _call(index, lib.tqb_paged_attention_rows, self._c, p, _want("cu", cu, torch.int32, (requests + 1,), index), n)
        return out


class PagedPqoCache:
    """A paged cache of all layers: pages, block tables, lengths and the list of free pages of up to `max_requests` running
    requests.  The counterpart of PqoCache (src/cache/pqo.rs:21-236) for requests of different lengths.

        step = cache.plan(new_tokens, capacity)                # once a step
        q = cache.append_rope(layer, rope, q, k, v, step)      # each layer
        out = cache.decode_tokens(layer, q, step, att).fused   # of the requests that bring one token
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
        self.failed = torch.zeros(1, dtype=torch.int32, device=dev)   # status of the last plan or release that did not fit
        self._scratch = {}

    def plan(self, new_tokens, capacity):
        """Pages, slots and positions for new_tokens [max_requests] int32 of each request; `step.check()` tells whether
        they fitted.  The step's kv_lens and state are the cache's own and go on with its next plan."""
        return paged_plan(self.seq_lens, new_tokens, self.block_table, self.free_pages, self.state, self.page_size, capacity,
                          kv_lens=self.seq_lens, state_out=self.state, failed=self.failed)

    def check(self):
        """Raises if any plan or release since the last check did not fit, those of replayed graphs included; waits for the
        device.  A step that did not fit has stored nothing."""
        status = int(torch.where(self.failed[0] != 0, self.failed[0], self.state[2]))
        if status:
            self.failed.zero_()
            self.state[2] = 0
        _check_plan(status)

    def release(self, mask):
        """Ends the requests with mask[r] (bool or u8 [max_requests]); their rows may be used by new ones.  Pages that others
        hold too stay theirs."""
        paged_release(mask, self.seq_lens, self.block_table, self.free_pages, self.state, self.page_size)

    def append(self, layer, k, v, step):
        self._layer(layer).append(k, v, step.slots[: k.shape[0]])

    def append_rope(self, layer, rope, q, k, v, step, q_out=None):
        n = k.shape[0]
        return self._layer(layer).append_rope(rope, q, k, v, step.positions[:n], step.slots[:n], q_out=q_out)

    def dequantize(self, layer, slots, dtype=torch.float32):
        return self._layer(layer).dequantize(slots, dtype)

    def decode(self, layer, q, step, config, out=None, scratch=None):
        """Attention of q [max_requests, query heads, dim] over everything stored, row r being request r's: DecodeOutput with
        `fused` set.  (The rows that append_rope returns are the step's tokens, which is something else as soon as a request
        is idle: they go to decode_tokens.)
        Without `scratch` the cache keeps one for each stream, and a call that is being captured gets its own."""
        return self._decode(layer, q, step, config, out, scratch, None)

    def decode_tokens(self, layer, q, step, config, out=None, scratch=None):
        """The same for the step's tokens: q [tokens, query heads, dim] as append_rope returns it, padding behind the last
        token included.  Rows of requests that bring one token are computed; of other rows see PagedLayer.attend."""
        return self._decode(layer, q, step, config, out, scratch, step.cu)

    def _decode(self, layer, q, step, config, out, scratch, cu):
        at = self._layer(layer)
        if scratch is None:
            stream = _eager_stream(at.index)
            if stream is not None:
                scratch = self._scratch.get(stream)
                if scratch is None:
                    scratch = self._scratch[stream] = at.attend_scratch(q.shape[1])
        return DecodeOutput(fused=at.attend(q, self.block_table, step.kv_lens, config.softmax_scale, out=out, scratch=scratch, cu=cu))

    def _layer(self, layer):
        if not 0 <= layer < len(self.layers):
            check(4)
        return self.layers[layer]

    def memory_usage(self):
        return sum(t.numel() * t.element_size() for x in self.layers for t in x.tensors)
