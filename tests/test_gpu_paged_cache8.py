"""GPU: a text model over a paged cache of 8-bit codes, against the same model over bf16 pages.

Layer 0's keys and values do not depend on the cache: they are the bf16 ones, quantised.  Values to
the bit; keys are turned by angles that were rounded finer than the bf16 pages', so that some are
the next bf16 number, 2^-7 off at most: int8's then differ by that, one scale, and by one for each
side's own rounding after its scale has grown; e4m3's by 2^-7 of the value and 2^-4 for each side.
What comes after them: an e4m3 row is off by 2^-4 of each value at most, evenly spread 2^-4 /
sqrt(3) or less by the 2-norm, 0.036; an int8 row by half a scale, 2^-7 of the block's largest
value, which is at most 6 times the 2-norm's mean here: 0.047 / sqrt(3) = 0.027.  The output's
values have that once, and its weights once more: scores are scale q.dk, with rows of norm sqrt(128)
off by 0.036 sqrt(128) in all and scale 128^-1/2, by 0.036 |q| / sqrt(128), a random walk.  Together
0.036 sqrt(2) of an attention's output by the 2-norm, which the residual stream only dilutes; two
layers in quadrature 0.072, and the bf16 steps' own 0.02: within 0.1."""

from __future__ import annotations

import pytest
import torch
from helpers import rel_err

import cache8_reference as ref8
from test_gpu_paged_cache import DEV, calls, text_model  # noqa: F401
from umic.paged_cache import PagedKVCache

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::FutureWarning"),
              pytest.mark.filterwarnings("ignore::UserWarning")]
TOL = 0.1


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_model_over_codes(kind, calls):  # noqa: F811
    m, _ = text_model()
    kw = dict(requests=4, pages=24, max_tokens=96, page_size=16)
    rows = PagedKVCache.for_model(m, **kw)
    codes = PagedKVCache.for_model(m, **kw, dtype=ref8.TYPES[kind])
    assert codes.arena.storage.dtype is ref8.TYPES[kind]
    shape = codes.arena.storage.shape[2:]
    model = [[torch.zeros(shape, dtype=torch.float64).numpy(),
              torch.ones(*shape[:2], shape[2] // 16, dtype=torch.float64).numpy()] for _ in range(2)]
    g = torch.Generator().manual_seed(1)
    steps = [([23, 1, 40, 16], None), (1, None), (1, None), ([1, 17, 1, 0], [None, 0, None, None]),
             ([3, 3, 1, 3], None), (1, [None, None, 0, 5]), (1, None)]
    with torch.no_grad():
        for new, keep in steps:
            lens = [new] * 4 if isinstance(new, int) else new
            ids = torch.randint(0, 512, (4, max(lens)), generator=g).to(DEV)
            out = []
            for c in (rows, codes):
                c.begin(new, keep=keep)
                out.append(m(input_ids=ids, position_ids=c.position_ids, past_key_values=c).last_hidden_state)
            assert rows.arena.lens == codes.arena.lens
            for r, n in enumerate(lens):
                if n:
                    assert rel_err(out[1][r, :n], out[0][r, :n]) <= TOL, (r, n)
            # layer 0, from the bf16 pages' rows: both arenas have the same table
            slots = [s for s in codes.step.slots.tolist() if s >= 0]
            want = []
            for which, (c8, scale) in zip((rows.arena.k(0), rows.arena.v(0)), model):
                flat = which.transpose(1, 2).flatten(0, 1).double().cpu().numpy()
                ref8.store(kind, c8, scale, flat[slots], slots)
                want.append(torch.tensor(ref8.values(c8, scale)))
            table = codes.arena.table.cpu()
            for i, (got, pool) in enumerate(zip(codes.arena.read(0), want)):
                scale = torch.tensor(model[i][1]).maximum(codes.arena.scales[0, i].double().cpu())
                scale = scale.repeat_interleave(16, 2)[..., None].expand(pool.shape)
                for r, n in enumerate(codes.arena.lens):
                    pages, s = (x[table[r, :-(-n // 16)].long()].transpose(0, 1).flatten(1, 2)[:, :n]
                                for x in (pool, scale))
                    off = (got[r, :, :n].double().cpu() - pages).abs()
                    tol = 3 * s if kind == "int8" else (2.0 ** -7 + 2.0 ** -3) * pages.abs() + 2.0 ** -8 * s
                    assert (off <= (tol if i == 0 else 0)).all(), (r, i)
                    assert not got[r, :, n:].any()
    both = 2 * len(steps)
    assert calls["umic_cache8_append_bf16"] == calls["umic_cache8_attention_bf16"] == both
    assert calls["umic_axial_rope_append_bf16"] == calls["umic_cache_attention_bf16"] == both
    assert calls["umic_cache8_read_bf16"] == len(steps)
    codes.reset()
    assert codes.arena.kv_len.tolist() == [0] * 4 and codes.arena.free == 24
