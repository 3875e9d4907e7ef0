"""The serving step over a paged key-value cache: ``assign``, ``store``, ``attend``.

Library operators of libemmyb200.so (include/emmy_b200.h states each in full) on torch tensors, with run-time sizes: one
step of a server calls ``assign`` once (pages and slots for the step's new tokens, from the requests' lengths), and in
each layer ``store`` (norm and rotation of the new queries and keys; keys and values into their slots) and ``attend``
(one new token of each request over its pages). Prompts' own rows go through the attention family.

Calls run on the current stream of the tensors' device, which need not be the current one, read nothing back and may be
captured into a CUDA graph. Arguments that the host can judge are refused with ``driver.EmbError`` (code -2). There is no
gradient: outputs are not part of a graph.
"""

from __future__ import annotations

import struct
from typing import NamedTuple

import torch

from . import driver

# the structures of include/emmy_b200.h, field by field
_CACHE = "QQ 3q 3q iiii i ff i"
_ASSIGN = struct.Struct("@ QQQQQQQQQQQ q iiii i i".replace(" ", ""))
_STORE = struct.Struct(("@ QQQQQQQQQ" + _CACHE + "2q 2q 2q 2q ii i i i i f i").replace(" ", ""))
_ATTEND = struct.Struct(("@ QQQQQQ" + _CACHE + "2q 2q q q ii i i i f").replace(" ", ""))

_CODE = {torch.float8_e4m3fn: 0, torch.float16: 1, torch.bfloat16: 2}
_BYTES = {0: 1, 1: 2, 2: 2}


class Assigned(NamedTuple):
    """What ``assign`` returns, all int32 tensors on the device."""
    slots: torch.Tensor
    positions: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor
    free_head: torch.Tensor
    report: torch.Tensor


def _refuse(text: str):
    raise driver.EmbError(-2, text)


def _call(entry, device: int, packed: bytes) -> None:
    """One call on the current stream of ``device``."""
    if device < 0:
        _refuse("the tensors are not on a CUDA device: the kernels run on the GPU only")
    if torch.cuda.current_device() == device:
        code = entry(packed, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            code = entry(packed, torch._C._cuda_getCurrentRawStream(device))
    if code:
        driver.check(code)


def _same_device(who: str, device: int, *tensors) -> None:
    for t in tensors:
        if t is not None and t.get_device() != device:
            _refuse(f"{who}: the tensors are on different devices")


def _int32(who: str, name: str, t, shape) -> None:
    if t.dtype is not torch.int32 or t.shape != shape or not t.is_contiguous():
        _refuse(f"{who}: {name} is a contiguous int32 tensor of {list(shape)}, not {t.dtype} {list(t.shape)}")


def _rows(who: str, name: str, t, dtype, heads, dim, count) -> tuple:
    """The strides of [rows, heads, dim] whose last dimension is contiguous."""
    if t.dtype is not dtype or t.shape != (count, heads, dim):
        _refuse(f"{who}: {name} is {dtype} [{count}, {heads}, {dim}], not {t.dtype} {list(t.shape)}")
    a, b, c = t.stride()
    if c != 1:
        _refuse(f"{who}: the last dimension of {name} is not contiguous")
    # a dimension of one has any stride
    return a if count > 1 else 0, b if heads > 1 else 0


def _cache(who: str, k, v, dtype, k_scale, v_scale) -> tuple:
    """(pages, page size, key heads, dim, the packed fields of emb_paged_cache_t)."""
    if k.dim() != 4 or k.shape != v.shape or k.dtype is not v.dtype:
        _refuse(f"{who}: key and value pages are two tensors [pages, page size, key heads, dim] of one type")
    code = _CODE.get(k.dtype)
    if code is None or (code and k.dtype is not dtype):
        _refuse(f"{who}: pages of {k.dtype} under queries of {dtype}: the same 16-bit type, or float8_e4m3fn")
    pages, size, heads, dim = k.shape
    ks, vs = k.stride(), v.stride()
    if ks[3] != 1 or vs[3] != 1:
        _refuse(f"{who}: the last dimension of the pages is not contiguous")
    if not code:
        pass
    elif k_scale != 1.0 or v_scale != 1.0:
        _refuse(f"{who}: scales belong to a float8_e4m3fn cache")
    if pages <= 1 or size <= 1 or heads <= 1:
        one = (pages > 1, size > 1, heads > 1)
        ks, vs = (tuple(s if many else 0 for s, many in zip(st, one)) for st in (ks, vs))
    return pages, size, heads, dim, (k.data_ptr(), v.data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], pages, size, heads, dim,
                                     code, k_scale, v_scale, 0)


def assign(cached, fresh, table, free_pages, free_head, page_size: int, tokens: int, out=None) -> Assigned:
    """Pages and slots of one step's new tokens (emb_paged_assign).

    ``cached``, ``fresh`` [requests]: tokens in the cache, and new ones. ``table`` [requests, width]: page ids, updated in
    place. ``free_pages`` [n] are handed out from entry ``free_head`` [1] on. ``tokens``: the step's rows, at least as
    many as there are new tokens. All int32. Returns slots and positions [tokens] (-1 and 0 behind the last request),
    starts [requests + 1], lengths [requests], free_head [1] and report [4] (pages taken, requests refused, rows wanted
    beyond ``tokens``, rows wanted); ``out``: these six tensors, to be written instead of new ones. A request whose tokens
    fit neither its table row nor the step nor the free pages is refused whole: slots -1, length and table as they were.
    """
    if cached.dim() != 1 or table.dim() != 2 or free_pages.dim() != 1:
        _refuse("assign: cached, fresh [requests], table [requests, width], free_pages [n]")
    requests, width = cached.shape[0], table.shape[1]
    _int32("assign", "cached", cached, (requests,))
    _int32("assign", "fresh", fresh, (requests,))
    _int32("assign", "free_pages", free_pages, free_pages.shape)
    _int32("assign", "free_head", free_head, (1,))
    if table.dtype is not torch.int32 or table.shape[0] != requests or (width > 1 and table.stride(1) != 1):
        _refuse(f"assign: table is an int32 tensor [{requests}, width] with contiguous rows")
    device = cached.get_device()
    if out is None:
        new = lambda n: torch.empty(n, dtype=torch.int32, device=cached.device)  # noqa: E731
        if tokens < 0:
            _refuse("assign: tokens is negative")
        out = Assigned(new(tokens), new(tokens), new(requests + 1), new(requests), new(1), new(4))
    else:
        out = Assigned(*out)
        for name, t, n in zip(Assigned._fields, out, (tokens, tokens, requests + 1, requests, 1, 4)):
            _int32("assign", "out." + name, t, (n,))
    _same_device("assign", device, fresh, table, free_pages, free_head, *out)
    _call(driver.library().emb_paged_assign, device, _ASSIGN.pack(
        cached.data_ptr(), fresh.data_ptr(), table.data_ptr(), free_pages.data_ptr(), free_head.data_ptr(), out[0].data_ptr(),
        out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), out[4].data_ptr(), out[5].data_ptr(),
        table.stride(0) if requests > 1 else width, requests, width, free_pages.shape[0], page_size, tokens, 0))
    return out


def store(q, k, v, k_pages, v_pages, slots, positions, rope=None, q_weight=None, k_weight=None, eps: float = 1e-6,
          interleaved: bool = False, k_scale: float = 1.0, v_scale: float = 1.0, out=None):
    """Norm and rotation of new queries and keys; keys and values into their slots (emb_paged_store). Returns the queries.

    ``q`` [tokens, heads, dim], ``k`` and ``v`` [tokens, key heads, dim], f16 or bf16 (views of one projection's output
    will do). Pages [pages, page size, key heads, dim] of the same type or float8_e4m3fn (value = code * scale), in any
    order of the first three dimensions. ``slots``, ``positions`` [tokens] int32; a slot of -1 stores nothing. ``rope``
    [positions, rot] f32: rot/2 cosines, then rot/2 sines; pairs (j, j + rot/2), or (2j, 2j + 1) where ``interleaved``.
    ``q_weight``, ``k_weight`` [dim]: y = x / sqrt(mean(x^2) + eps) * weight over each head; None: no norm. ``out`` may
    be ``q``.
    """
    if q.dim() != 3:
        _refuse("store: q is [tokens, heads, dim]")
    tokens, heads, dim = q.shape
    dtype = q.dtype
    _, _, kv_heads, page_dim, cache = _cache("store", k_pages, v_pages, dtype, k_scale, v_scale)
    if page_dim != dim:
        _refuse(f"store: heads of {dim}, pages of {page_dim}")
    q_stride = _rows("store", "q", q, dtype, heads, dim, tokens)
    k_stride = _rows("store", "k", k, dtype, kv_heads, dim, tokens)
    v_stride = _rows("store", "v", v, dtype, kv_heads, dim, tokens)
    _int32("store", "slots", slots, (tokens,))
    rot = rope_rows = rope_at = positions_at = 0
    if rope is not None:
        if rope.dtype is not torch.float32 or rope.dim() != 2 or not rope.is_contiguous():
            _refuse("store: rope is a contiguous float32 tensor [positions, rot]")
        rope_rows, rot = rope.shape
        _int32("store", "positions", positions, (tokens,))
        rope_at, positions_at = rope.data_ptr(), positions.data_ptr()
    weights_at = []
    for name, w in (("q_weight", q_weight), ("k_weight", k_weight)):
        if w is not None and (w.dtype is not dtype or w.shape != (dim,) or not w.is_contiguous()):
            _refuse(f"store: {name} is a contiguous {dtype} tensor [{dim}]")
        weights_at.append(0 if w is None else w.data_ptr())
    if out is None:
        out = torch.empty(tokens, heads, dim, dtype=dtype, device=q.device)
    out_stride = _rows("store", "out", out, dtype, heads, dim, tokens)
    device = q.get_device()
    _same_device("store", device, k, v, k_pages, v_pages, slots, positions if rot else None, rope, q_weight, k_weight, out)
    _call(driver.library().emb_paged_store, device, _STORE.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), slots.data_ptr(), positions_at, rope_at, *weights_at, *cache,
        *q_stride, *k_stride, *v_stride, *out_stride, tokens, heads, _CODE[dtype], rot, rope_rows, interleaved, eps, 0))
    return out


def attend(q, k_pages, v_pages, table, lengths, scale: float | None = None, window: int = 0, k_scale: float = 1.0,
           v_scale: float = 1.0, out=None, lse=None):
    """Attention of one new token of each request over its pages (emb_paged_attend). Returns [requests, heads, dim].

    ``q`` [requests, heads, dim] f16 or bf16; ``heads`` a multiple of the pages' key heads, query head h reads key head
    h // (heads // key heads). ``table`` [requests, width] and ``lengths`` [requests] int32: key j of request b is token
    j % page size of page table[b, j // page size], j < lengths[b], the new token's own among them; ``window``: only the
    last so many (0: all). ``scale``: 1 / sqrt(dim) where None. A request of length 0 gives 0. ``lse`` [requests, heads]
    f32: written with the logarithm of the sum of exponentials.
    """
    if q.dim() != 3:
        _refuse("attend: q is [requests, heads, dim]")
    requests, heads, dim = q.shape
    dtype = q.dtype
    _, _, _, page_dim, cache = _cache("attend", k_pages, v_pages, dtype, k_scale, v_scale)
    if page_dim != dim:
        _refuse(f"attend: heads of {dim}, pages of {page_dim}")
    q_stride = _rows("attend", "q", q, dtype, heads, dim, requests)
    _int32("attend", "lengths", lengths, (requests,))
    if table.dim() != 2 or table.dtype is not torch.int32 or table.shape[0] != requests or (table.shape[1] > 1 and table.stride(1) != 1):
        _refuse(f"attend: table is an int32 tensor [{requests}, width] with contiguous rows")
    if out is None:
        out = torch.empty(requests, heads, dim, dtype=dtype, device=q.device)
    out_stride = _rows("attend", "out", out, dtype, heads, dim, requests)
    lse_at = 0
    if lse is not None:
        if lse.dtype is not torch.float32 or lse.shape != (requests, heads) or not lse.is_contiguous():
            _refuse(f"attend: lse is a contiguous float32 tensor [{requests}, {heads}]")
        lse_at = lse.data_ptr()
    device = q.get_device()
    _same_device("attend", device, k_pages, v_pages, table, lengths, out, lse)
    lib = driver.library()
    fields = [q.data_ptr(), out.data_ptr(), lse_at, table.data_ptr(), lengths.data_ptr(), 0, *cache, *q_stride, *out_stride,
              table.stride(0), 0, requests, heads, table.shape[1], _CODE[dtype], window, dim ** -0.5 if scale is None else scale]
    if device >= 0:
        with torch.cuda.device(device):
            need = lib.emb_paged_attend_workspace(_ATTEND.pack(*fields))
        if need < 0:
            driver.check(need)
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device)
        fields[5], fields[-7] = workspace.data_ptr(), need
    _call(lib.emb_paged_attend, device, _ATTEND.pack(*fields))
    return out
