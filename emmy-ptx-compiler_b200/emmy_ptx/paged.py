"""The serving step over a paged key-value cache: ``assign``, ``store``, ``attend``.

Library operators of libemmyb200.so (include/emmy_b200.h states each in full) on torch tensors, with run-time sizes: one
step of a server calls ``assign`` once (pages and slots for the step's new tokens, from the requests' lengths), and in
each layer ``store`` (norm and rotation of the new queries and keys; keys and values into their slots) and ``attend``
(one new token of each request over its pages). There is no attention of several new tokens of a request over its pages: a
prompt's own goes through the attention family, from keys that the caller norms and rotates as ``store`` does (it returns the
queries only), and a prompt piece on top of cached tokens has none.

Calls run on the current stream of the tensors' device, which need not be the current one, read nothing back and may be
captured into a CUDA graph. Arguments that the host can judge are refused with ``driver.EmbError`` (code -2). There is no
gradient: a tensor that requires one is refused where gradients are on, and so is one with a tangent (forward mode).
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from . import driver

_native = None


def _load():
    """The binding (csrc/binding/paged_torch.cpp), loaded once. Built by ``__graft_entry__.build()``."""
    global _native
    if _native is None:
        driver.library()
        try:
            from . import _paged
        except ImportError as e:
            raise driver.EmbError(-100, f"emmy_ptx/_paged.so cannot be loaded ({e}): build it first (python -c 'import __graft_entry__ as g; g.build()')") from e
        _paged.init(driver.EmbError)
        _native = _paged
    return _native


class Assigned(NamedTuple):
    """What ``assign`` returns, all int32 tensors on the device."""
    slots: torch.Tensor
    positions: torch.Tensor
    starts: torch.Tensor
    lengths: torch.Tensor
    free_head: torch.Tensor
    report: torch.Tensor


def assign(cached, fresh, table, free_pages, free_head, page_size: int, tokens: int, out=None) -> Assigned:
    """Pages and slots of one step's new tokens (emb_paged_assign).

    ``cached``, ``fresh`` [requests]: tokens in the cache, and new ones. ``table`` [requests, width]: page ids, updated in
    place. ``free_pages`` [n] are handed out from entry ``free_head`` [1] on. ``tokens``: the step's rows, at least as
    many as there are new tokens. All int32. Returns slots and positions [tokens] (-1 and 0 behind the last request),
    starts [requests + 1], lengths [requests], free_head [1] and report [4] (pages taken, requests refused, rows wanted
    beyond ``tokens``, rows wanted); ``out``: these six tensors, to be written instead of new ones (in memory that
    is none of the inputs' and not shared). A request whose tokens
    fit neither its table row nor the step nor the free pages is refused whole: slots -1, length and table as they were.
    """
    if out is not None and type(out) is not Assigned:
        out = Assigned(*out)
    got = (_native or _load()).assign(cached, fresh, table, free_pages, free_head, page_size, tokens, out)
    return got if out is not None else Assigned._make(got)


def store(q, k, v, k_pages, v_pages, slots, positions, rope=None, q_weight=None, k_weight=None, eps: float = 1e-6,
          interleaved: bool = False, k_scale: float = 1.0, v_scale: float = 1.0, out=None):
    """Norm and rotation of new queries and keys; keys and values into their slots (emb_paged_store). Returns the queries.

    ``q`` [tokens, heads, dim], ``k`` and ``v`` [tokens, key heads, dim], f16 or bf16 (views of one projection's output
    will do). Pages [pages, page size, key heads, dim] of the same type or float8_e4m3fn (value = code * scale), in any
    order of the first three dimensions. ``slots``, ``positions`` [tokens] int32; a slot of -1 stores nothing. ``rope``
    [positions, rot] f32: rot/2 cosines, then rot/2 sines; pairs (j, j + rot/2), or (2j, 2j + 1) where ``interleaved``.
    ``q_weight``, ``k_weight`` [dim]: y = x / sqrt(mean(x^2) + eps) * weight over each head; None: no norm. ``out`` may
    be ``q``; other memory that the call reads, or writes elsewhere, is refused as an output.
    """
    return (_native or _load()).store(q, k, v, k_pages, v_pages, slots, positions, rope, q_weight, k_weight, eps, interleaved, k_scale, v_scale, out)


def attend(q, k_pages, v_pages, table, lengths, scale: float | None = None, window: int = 0, k_scale: float = 1.0,
           v_scale: float = 1.0, out=None, lse=None):
    """Attention of one new token of each request over its pages (emb_paged_attend). Returns [requests, heads, dim].

    ``q`` [requests, heads, dim] f16 or bf16; ``heads`` a multiple of the pages' key heads, query head h reads key head
    h // (heads // key heads). ``table`` [requests, width] and ``lengths`` [requests] int32: key j of request b is token
    j % page size of page table[b, j // page size], j < lengths[b], the new token's own among them; ``window``: only the
    last so many (0: all). ``scale``: 1 / sqrt(dim) where None. A request of length 0 gives 0. ``lse`` [requests, heads]
    f32: written with the logarithm of the sum of exponentials. ``out`` may be ``q``; other memory that the call reads is
    refused as an output.
    """
    return (_native or _load()).attend(q, k_pages, v_pages, table, lengths, scale, window, k_scale, v_scale, out, lse)
