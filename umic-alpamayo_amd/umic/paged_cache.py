"""A paged KV cache: requests of different lengths in one pool, for a text model
that decodes them together.

Storage.  ``PagedArena`` holds every layer's pages, ``[layers, 2, pages, kv_heads,
page_size, head_dim]`` (a layer's keys and values are what the kernels of
``umic.kernels.axial`` and ``umic.kernels.attention`` take), and one set of block
tables, lengths and free pages for all layers, on the device, with the lengths
mirrored on the host.

A step.  ``cache.begin(new)`` plans it: the tokens each request drops and gets,
their pages, slots and positions (``paged.plan_pages``).  The model's forward is
then called as usual, ``input_ids`` [requests, S] with ``past_key_values=cache``: an
attention patched by ``umic.integrate.fuse_kv_rope`` norms and rotates q and k into
the pages in one launch and attends over them in another.

    cache = PagedKVCache.for_model(lm, requests=16, pages=4096, max_tokens=8192)
    cache.begin([len(p) for p in prompts])             # right-padded prompts
    lm(input_ids=prompts, position_ids=cache.position_ids, past_key_values=cache)
    cache.begin(1)                                     # a token each
    cache.begin(1, keep=[0, None, ...])                # request 0 starts anew

Positions come from the plan (the token's place in its request plus ``delta``) or
from the caller, through ``begin``, as [axes, requests, S] (image grids); position ids
of the forward that differ from them are refused.  Numerics are ``axial``'s and
``attention``'s: fp32 with one rounding, where the in-place cache repeats the eager
chain's roundings.

No counterpart in the reference, whose cache is of one batch of equal lengths
(src/umic/cache.py:25-160).
"""

from __future__ import annotations

from typing import Sequence

import torch
from transformers.cache_utils import DynamicCache

from umic.kernels import attention, axial, paged


_ALL = 2 ** 31 - 1  # keep: whatever is held


class PagedArena:
    """Pages of ``layers`` layers that ``requests`` requests share.

    max_tokens: tokens that one request can hold.

    ``lens`` and ``free`` mirror the device's lengths and free pages, and ``plan``
    refuses by them what does not fit.  Steps that go past ``plan`` (a captured
    ``paged.plan_pages`` on these tensors, replayed) leave them behind: ``sync`` reads
    them again, before the next ``plan``.  The tensors stay the same ones; a step's
    kv_len and cursor are the arena's.
    """

    def __init__(self, layers: int, requests: int, pages: int, heads: int, page_size: int,
                 head_dim: int, max_tokens: int, device: torch.device | str = "cuda") -> None:
        if min(layers, requests, pages, heads, max_tokens) <= 0:
            raise ValueError(f"PagedArena: bad geometry layers={layers} requests={requests} "
                             f"pages={pages} heads={heads} max_tokens={max_tokens}")
        if not paged.page_size_ok(page_size) or head_dim not in attention.HEAD_DIMS:
            raise ValueError(f"PagedArena: page_size {page_size} (powers of two from 16), "
                             f"head_dim {head_dim} (one of {attention.HEAD_DIMS})")
        self.page_size, self.requests, self.pages = page_size, requests, pages
        width = -(-max_tokens // page_size)
        self.max_tokens = width * page_size
        self.storage = torch.empty(layers, 2, pages, heads, page_size, head_dim,
                                   dtype=torch.bfloat16, device=device)
        ints = dict(dtype=torch.int32, device=device)
        self.table = torch.zeros(requests, width, **ints)
        self.ring = torch.arange(pages, **ints)
        self.cursor = torch.tensor([0, pages, 0, 0], **ints)
        self.kv_len = torch.zeros(requests, **ints)
        self.lens = [0] * requests  # kv_len, on the host
        self.free = pages

    def k(self, layer: int) -> torch.Tensor:
        return self.storage[layer, 0]

    def v(self, layer: int) -> torch.Tensor:
        return self.storage[layer, 1]

    def _ints(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(values, dtype=torch.int32, device=self.kv_len.device)

    def plan(self, new: Sequence[int], keep: Sequence[int | None] | None = None,
             delta: Sequence[int] | None = None):
        """One step: request r keeps its first keep[r] tokens (None: all) and gets
        new[r]; (PageStep, new as a device vector).  Raises, and changes nothing,
        where the pages do not suffice."""
        n, ps = self.requests, self.page_size
        if len(new) != n or any(x is not None and len(x) != n for x in (keep, delta)):
            raise ValueError(f"PagedArena: a step is of {n} requests")
        if min(new) < 0:
            raise ValueError(f"PagedArena: new tokens {list(new)}")
        kept = self.lens if keep is None else [
            held if k is None else max(0, min(k, held)) for k, held in zip(keep, self.lens)]
        lens = [k + x for k, x in zip(kept, new)]
        free = self.free + sum(-(-held // ps) - -(-x // ps) for held, x in zip(self.lens, lens))
        if max(lens) > self.max_tokens:
            raise RuntimeError(f"paged cache overflow: request {lens.index(max(lens))} of "
                               f"{max(lens)} tokens > {self.max_tokens}")
        if free < 0:
            raise RuntimeError(f"paged cache overflow: {-free} pages of {ps} tokens are missing")
        row = max(max(new), 1)
        fresh = self._ints(new)
        # lengths and queue in place: captured steps hold their addresses
        starts = fresh.new_empty(n + 1)
        slots, positions = fresh.new_empty(2, n * row, dtype=torch.int64)
        step = paged.plan_pages(
            self.kv_len, fresh, self.table, self.ring, self.cursor, ps, n * row,
            keep=None if keep is None else self._ints(
                [_ALL if k is None else max(0, min(k, _ALL)) for k in keep]),
            delta=None if delta is None else self._ints(delta), row=row,
            out=paged.PageStep(self.kv_len, self.cursor, starts, slots, positions))
        self.lens, self.free = lens, free
        return step, fresh

    def sync(self) -> None:
        """lens and free as the device has them.  Raises where the last step was refused
        there (it changed nothing: its tokens are not in the pages)."""
        _, self.free, _, status = self.cursor.tolist()
        self.lens = self.kv_len.tolist()
        if status != paged.PLAN_OK:
            raise RuntimeError(f"paged cache: the last step was refused "
                               f"({paged.REFUSALS[status]})")


def _refuse(module, args, kwargs):
    """Forward pre-hook of a text model: a ``PagedKVCache`` goes without a mask, and with
    the positions of its step.  What transformers makes of no mask, where it cannot look
    at the lengths (a capture), is then known to hold nothing."""
    mask = kwargs.get("attention_mask", args[1] if len(args) > 1 else None)
    positions = kwargs.get("position_ids", args[2] if len(args) > 2 else None)
    cache = kwargs.get("past_key_values", args[3] if len(args) > 3 else None)
    if isinstance(cache, PagedKVCache):
        tokens = kwargs.get("input_ids", args[0] if args else None)
        if tokens is None:
            tokens = kwargs.get("inputs_embeds", args[4] if len(args) > 4 else None)
        if positions is not None and cache.planned(tokens) and not cache.turns_by(positions):
            raise ValueError("PagedKVCache: position_ids are not those of its step, which its "
                             "attention turns by: give them to begin(), and the forward "
                             "cache.position_ids")
        if mask is not None:
            raise ValueError("PagedKVCache: its lengths say which tokens are seen; pass no "
                             "attention_mask (begin() takes the prompts' lengths)")
        cache.unmasked = True


class PagedKVCache(DynamicCache):
    """A ``PagedArena`` as the cache of a transformers text model whose attention
    ``umic.integrate.fuse_kv_rope`` has patched.

    rotary: the plan of the arena's head size, on its device.
    query_heads: of the model, if ``begin`` is to refuse a step that the attention does
        not take.
    """

    def __init__(self, arena: PagedArena, rotary: axial.AxisPlan,
                 query_heads: int | None = None) -> None:
        super().__init__()
        dim = arena.storage.shape[-1]
        if rotary.head_dim != dim or rotary.turn.device != arena.storage.device:
            raise ValueError(f"PagedKVCache: a rotary plan of heads of {rotary.head_dim} on "
                             f"{rotary.turn.device} for pages of {dim} on {arena.storage.device}")
        self.arena, self.rotary, self.query_heads = arena, rotary, query_heads
        self.step: paged.PageStep | None = None
        self.tokens = 0  # of a request, in the open step
        self.unmasked = False  # the running forward was called without a mask
        self._before = [0] * arena.requests
        self._fresh: torch.Tensor | None = None
        self._positions: torch.Tensor | None = None

    @classmethod
    def for_model(cls, lm: torch.nn.Module, requests: int, pages: int, max_tokens: int,
                  page_size: int = 64) -> "PagedKVCache":
        """A cache for the text model ``lm`` (``layers`` with ``self_attn``, and
        ``rotary_emb``)."""
        attn = lm.layers[0].self_attn
        weight = attn.k_proj.weight
        heads = weight.shape[0] // attn.head_dim
        arena = PagedArena(len(lm.layers), requests, pages, heads, page_size, attn.head_dim,
                           max_tokens, weight.device)
        if getattr(lm, "_umic_paged_hook", None) is None:
            lm._umic_paged_hook = lm.register_forward_pre_hook(_refuse, with_kwargs=True)
        return cls(arena, axial.AxisPlan.rotary(lm.rotary_emb),
                   attn.q_proj.weight.shape[0] // attn.head_dim)

    def begin(self, new: int | Sequence[int], positions: torch.Tensor | None = None,
              keep: Sequence[int | None] | None = None, delta: Sequence[int] | None = None) -> None:
        """Plan the next forward: its tokens of each request (an int: as many of all),
        right-padded to the longest.  positions: [axes, requests, S] int64, else the
        plan's own plus ``delta``.  What does not fit is refused here, and changes
        nothing.  The forward has to be run before the next step: it writes the rows
        that the plan has counted."""
        ar = self.arena
        same = isinstance(new, int)
        new = [new] * ar.requests if same else list(new)
        tokens = max(max(new), 1)
        want = (self.rotary.axes, ar.requests, tokens)
        if positions is not None and tuple(positions.shape) != want:
            raise ValueError(f"PagedKVCache: positions {tuple(positions.shape)}, not {want}: a row "
                             "for each axis of the rotary plan (no row of text positions ahead of "
                             "them), requests, tokens")
        if positions is not None and (positions.dtype is not torch.int64
                                      or positions.device != ar.storage.device):
            raise ValueError(f"PagedKVCache: positions must be int64 on {ar.storage.device}, got "
                             f"{positions.dtype} on {positions.device}")
        heads, dim = ar.storage.shape[3], ar.storage.shape[5]
        if self.query_heads and not attention.max_requests(tokens, self.query_heads, heads, dim,
                                                           ar.max_tokens):
            raise ValueError(f"PagedKVCache: {tokens} new tokens of {self.query_heads} heads over up "
                             f"to {ar.max_tokens} keys are too many for one launch")
        self.step, fresh = ar.plan(new, keep, delta)
        self.tokens, self.unmasked = tokens, False
        self._before = [n - x for n, x in zip(ar.lens, new)]
        # all rows are tokens: the attention needs no lengths of the new ones
        self._fresh = None if min(new) == tokens else fresh
        axes = self.rotary.axes
        self._positions = (self.step.positions.expand(axes, -1) if positions is None
                           else positions.reshape(positions.shape[0], -1))

    @property
    def position_ids(self) -> torch.Tensor:
        """The open step's positions, [axes, requests, S], as the model takes them."""
        return self._positions.reshape(-1, self.arena.requests, self.tokens)

    def planned(self, tokens: torch.Tensor | None) -> bool:
        """Whether a forward's input is the open step's by its shape ([requests, S, ..]);
        ``attend`` refuses others."""
        return (self.step is not None and tokens is not None
                and tuple(tokens.shape[:2]) == (self.arena.requests, self.tokens))

    def turns_by(self, positions: torch.Tensor) -> bool:
        """Whether a forward's position ids are the open step's for its tokens: this
        object's own without a look at them, others by their values (a wait for the
        device, and no for a capture).  Those of fewer axes or requests count for all,
        and a row of text positions ahead of the axes' does not count."""
        mine = self.position_ids
        if positions.dim() == 3 and positions.shape[0] == mine.shape[0] + 1:
            positions = positions[1:]
        if (positions.data_ptr() == mine.data_ptr() and positions.dtype is mine.dtype
                and positions.shape == mine.shape and positions.stride() == mine.stride()):
            return True
        if (positions.device != mine.device or positions.dim() > 3
                or any(n not in (1, m) for n, m in zip(positions.shape[::-1], mine.shape[::-1]))
                or torch.cuda.is_current_stream_capturing()):
            return False
        there = self.step.slots.view(mine.shape[1:]) >= 0
        return not bool(((positions != mine) & there).any())

    def attend(self, layer: int, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, norm,
               scale: float, causal: bool = True) -> torch.Tensor:
        """Append the step's k and v [requests, S, heads, D] to a layer's pages, rotated
        (and with ``norm = (q_w, k_w, eps)`` normed), and attend: [requests, S, Hq, D].
        Not causal: a request's new tokens see each other too."""
        B, S, Hq, D = q.shape
        ar = self.arena
        if self.step is None or B != ar.requests or S != self.tokens:
            raise RuntimeError(f"PagedKVCache: a forward of {B} x {S} tokens; begin() planned "
                               f"{ar.requests} x {self.tokens}")
        keys, values = ar.k(layer), ar.v(layer)
        flat = (t.reshape(B * S, -1, D) for t in (q, k, v))
        rot = axial.rotate_append(*flat, self._positions, self.rotary, self.step.slots, keys,
                                  values, norm)
        return attention.cache_attention(rot.view(B, S, Hq, D).transpose(1, 2), keys, values,
                                         ar.kv_len, table=ar.table, q_len=self._fresh,
                                         causal=causal, scale=scale)

    # -- what transformers asks of a cache -----------------------------------

    def update(self, key_states, value_states, layer_idx, *args, **kwargs):
        raise RuntimeError("PagedKVCache is read and written by attentions that "
                           "umic.integrate.fuse_kv_rope has patched, outside autograd")

    def get_seq_length(self, layer_idx: int = 0, cache_position=None) -> int:
        """Tokens that the longest request held before the open step."""
        return max(self._before)

    def get_mask_sizes(self, query_length, layer_idx: int = 0) -> tuple[int, int]:
        # the lengths say what is seen; a mask as of a prompt's own tokens is none
        n = query_length if isinstance(query_length, int) else query_length.shape[0]
        return n, 0

    def get_query_offset(self, layer_idx: int = 0) -> int:
        return 0

    def get_max_length(self, layer_idx=None) -> int:
        return self.arena.max_tokens

    get_max_cache_shape = get_max_length

    def crop(self, *args, **kwargs) -> None:
        raise RuntimeError("PagedKVCache: drop tokens with begin(..., keep=)")

    def reorder_cache(self, *args, **kwargs) -> None:
        raise RuntimeError("PagedKVCache: its requests stay where they are")

    batch_repeat_interleave = batch_select_indices = reorder_cache

    def sync(self) -> None:
        """``PagedArena.sync``, after replays of a captured step."""
        self.arena.sync()

    def reset(self) -> None:
        """Every request empty."""
        ar = self.arena
        ar.plan([0] * ar.requests, keep=[0] * ar.requests)
        self.step, self._before = None, [0] * ar.requests
