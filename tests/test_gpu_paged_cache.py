"""GPU: a text model over a paged cache, and the in-place cache's attention kernel in the model.

The reference is the unpatched model on the CPU, in bf16 with eager attention, each request by
itself on transformers' own cache.  Both round to bf16 after every operation, in other places
(about ten times a layer, 2^-9 of a value each, as a random walk 2^-7 over two layers): within
2e-2 by the 2-norm, the tolerance of this package's layer tests.
"""

from __future__ import annotations

import collections
import copy

import pytest
import torch
from helpers import rel_err

from umic import _lib, integrate
from umic.cache import InplaceKVCache
from umic.graph import DecodeGraphRunner
from umic.paged_cache import PagedKVCache

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::FutureWarning"),
              pytest.mark.filterwarnings("ignore::UserWarning")]
DEV = "cuda"
TOL = 2e-2


def text_model(kv_heads=2):
    from transformers.models.qwen3_vl.configuration_qwen3_vl import Qwen3VLTextConfig
    from transformers.models.qwen3_vl.modeling_qwen3_vl import Qwen3VLTextModel

    cfg = Qwen3VLTextConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=2,
                            num_attention_heads=4, num_key_value_heads=kv_heads, head_dim=128,
                            vocab_size=512,
                            rope_parameters={"rope_type": "default", "rope_theta": 1e6,
                                             "mrope_section": [24, 20, 20],
                                             "mrope_interleaved": True},
                            attn_implementation="sdpa")
    torch.manual_seed(0)
    m = Qwen3VLTextModel(cfg)
    with torch.no_grad():
        for name, p in m.named_parameters():
            if "norm" in name:
                p.copy_(1 + 0.1 * torch.randn_like(p))
    m = m.to(torch.bfloat16).eval()
    plain = copy.deepcopy(m)
    plain.config._attn_implementation = "eager"
    m = m.to(DEV)
    assert integrate.fuse_kv_rope(m) == 2
    return m, plain


@pytest.fixture
def calls(monkeypatch):
    log = collections.Counter()
    real = _lib.call

    def spy(name, *args):
        log[name] += 1
        return real(name, *args)

    monkeypatch.setattr(_lib, "call", spy)
    return log


def step_alone(plain, state, ids, pos):
    """One request's tokens by themselves: ids [n], pos [3, n]."""
    out = plain(input_ids=ids[None], position_ids=pos[:, None], past_key_values=state,
                use_cache=True)
    return out.last_hidden_state[0], out.past_key_values


def test_requests_of_different_lengths(calls):
    m, plain = text_model()
    c = PagedKVCache.for_model(m, requests=4, pages=24, max_tokens=96, page_size=16)
    g = torch.Generator().manual_seed(1)
    alone = [None] * 4
    steps = [([23, 1, 40, 16], None), (1, None), (1, None), ([1, 17, 1, 0], [None, 0, None, None]),
             ([3, 3, 1, 3], None), (1, [None, None, 0, 5]), (1, None)]
    with torch.no_grad():
        for new, keep in steps:
            c.begin(new, keep=keep)
            lens = [new] * 4 if isinstance(new, int) else new
            S = max(lens)
            ids = torch.randint(0, 512, (4, S), generator=g)
            pos = c.position_ids
            out = m(input_ids=ids.to(DEV), position_ids=pos, past_key_values=c).last_hidden_state
            assert out.shape == (4, S, 256)
            for r, n in enumerate(lens):
                if keep is not None and keep[r] is not None:
                    if keep[r] == 0:
                        alone[r] = None
                    else:
                        alone[r].crop(keep[r] - alone[r].get_seq_length())
                if n == 0:
                    continue
                held = 0 if alone[r] is None else alone[r].get_seq_length()
                assert pos[0, r, :n].tolist() == list(range(held, held + n))
                want, alone[r] = step_alone(plain, alone[r], ids[r, :n], pos[:, r, :n].cpu())
                assert rel_err(out[r, :n], want) <= TOL, (r, n)
                assert c.arena.lens[r] == held + n
            assert c.arena.kv_len.tolist() == c.arena.lens
            assert c.arena.cursor.tolist()[1::2] == [c.arena.free, 0]
    assert calls["umic_page_plan"] == len(steps)
    assert calls["umic_axial_rope_append_bf16"] == calls["umic_cache_attention_bf16"] == 2 * len(steps)
    c.reset()
    assert c.arena.kv_len.tolist() == [0] * 4 and c.arena.free == 24


def test_positions_of_an_image(calls):
    """Three different axes, given by the caller."""
    m, plain = text_model()
    c = PagedKVCache.for_model(m, requests=1, pages=8, max_tokens=96)
    g = torch.Generator().manual_seed(2)
    pos = torch.stack([torch.randint(0, 40, (1, 30), generator=g) for _ in range(3)])
    ids = torch.randint(0, 512, (1, 30), generator=g)
    with torch.no_grad():
        c.begin(30, positions=pos.to(DEV))
        out = m(input_ids=ids.to(DEV), position_ids=c.position_ids, past_key_values=c)
        want, state = step_alone(plain, None, ids[0], pos[:, 0])
        assert rel_err(out.last_hidden_state[0], want) <= TOL
        nxt = torch.randint(0, 512, (1, 1), generator=g)
        c.begin(1, delta=[11])
        assert c.position_ids.flatten().tolist() == [41] * 3
        out = m(input_ids=nxt.to(DEV), position_ids=c.position_ids, past_key_values=c)
        want, _ = step_alone(plain, state, nxt[0], torch.full((3, 1), 41))
        assert rel_err(out.last_hidden_state[0], want) <= TOL


def test_attention_without_norm_weights_and_refusals():
    """Head norms with a hook run as modules; a forward that was not planned, a mask and autograd
    are refused."""
    m, plain = text_model()
    c = PagedKVCache.for_model(m, requests=2, pages=8, max_tokens=64)
    ids = torch.randint(0, 512, (2, 9), generator=torch.Generator().manual_seed(3))
    seen = []
    handle = m.layers[0].self_attn.q_norm.register_forward_hook(lambda *a: seen.append(1))
    with torch.no_grad():
        c.begin(9)
        pos = c.position_ids
        out = m(input_ids=ids.to(DEV), position_ids=pos, past_key_values=c).last_hidden_state
        handle.remove()
        assert seen == [1]
        for r in range(2):
            want, _ = step_alone(plain, None, ids[r], pos[:, r].cpu())
            assert rel_err(out[r], want) <= TOL
        with pytest.raises(RuntimeError, match="planned"):
            m(input_ids=ids.to(DEV)[:, :3], position_ids=pos[..., :3], past_key_values=c)
        c.begin(1)
        with pytest.raises(ValueError, match="attention_mask"):
            m(input_ids=ids.to(DEV)[:, :1], attention_mask=torch.ones(2, 10, device=DEV),
              position_ids=c.position_ids, past_key_values=c)
        with pytest.raises(ValueError, match="attention_mask"):
            m.layers[0].self_attn(torch.zeros(2, 1, 256, dtype=torch.bfloat16, device=DEV),
                                  (None, None), torch.ones(2, 1, 1, 10, device=DEV),
                                  past_key_values=c)
    with pytest.raises(RuntimeError, match="outside autograd"):
        m(input_ids=ids.to(DEV)[:, :1], position_ids=c.position_ids, past_key_values=c)


def test_step_in_a_graph():
    """A decode step of all requests, captured: plan, layers and logits' input; every replay
    against an eager step on a cache of its own."""
    m, _ = text_model()
    g = torch.Generator().manual_seed(4)
    prompt = torch.randint(0, 512, (3, 20), generator=g).to(DEV)
    caches = []
    with torch.no_grad():
        for _ in range(2):
            c = PagedKVCache.for_model(m, requests=3, pages=12, max_tokens=64, page_size=16)
            c.begin([20, 5, 13])
            m(input_ids=prompt, position_ids=c.position_ids, past_key_values=c)
            caches.append(c)
        graphed, eager = caches
        ids = torch.zeros(3, 1, dtype=torch.long, device=DEV)
        eager.begin(1)   # library lazy initialisation outside the capture
        m(input_ids=ids, position_ids=eager.position_ids, past_key_values=eager)
        graphed.begin(1)
        m(input_ids=ids, position_ids=graphed.position_ids, past_key_values=graphed)
        from umic.kernels import paged

        ar = graphed.arena
        fresh = torch.ones(3, dtype=torch.int32, device=DEV)
        out = paged.PageStep(ar.kv_len, ar.cursor, *graphed.step[2:])
        graphed.step = out
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged.plan_pages(ar.kv_len, fresh, ar.table, ar.ring, ar.cursor, 16, 3, row=1, out=out)
            graphed._positions = out.positions.expand(3, -1)
            got = m(input_ids=ids, position_ids=graphed.position_ids,
                    past_key_values=graphed).last_hidden_state
        for _ in range(20):
            ids.copy_(torch.randint(0, 512, (3, 1), generator=g))
            eager.begin(1)
            want = m(input_ids=ids, position_ids=eager.position_ids,
                     past_key_values=eager).last_hidden_state
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert ar.kv_len.tolist() == eager.arena.lens


def test_decode_over_the_inplace_cache(calls):
    """fuse_cache_attention: a decode loop on an InplaceKVCache, the whole cache read where it
    lies."""
    from transformers.cache_utils import DynamicCache

    m, plain = text_model()
    assert integrate.fuse_cache_attention(m, dry_run=True) == 2
    assert not hasattr(m.layers[0].self_attn, "_umic_cache_attention")
    assert integrate.fuse_cache_attention(m) == 2
    g = torch.Generator().manual_seed(5)
    ids = torch.randint(0, 512, (1, 33), generator=g)
    pos = torch.arange(33).expand(3, 33)
    with torch.no_grad():
        want, state = step_alone(plain, None, ids[0], pos)
        prompt = DynamicCache()
        m2 = copy.deepcopy(plain).to(DEV)
        m2.config._attn_implementation = "eager"
        for layer, src in enumerate(state.layers):
            prompt.update(src.keys.to(DEV), src.values.to(DEV), layer)
        c = InplaceKVCache.from_dynamic(prompt, extra_tokens=16)
        for step in range(6):
            tok = torch.randint(0, 512, (1, 1), generator=g)
            p = torch.full((3, 1), 33 + step)
            out = m(input_ids=tok.to(DEV), position_ids=p[:, None].to(DEV), past_key_values=c)
            want, state = step_alone(plain, state, tok[0], p)
            assert rel_err(out.last_hidden_state[0], want) <= TOL
            assert c.get_seq_length() == 34 + step
            assert c.layers[0].keys.shape[2] == 34 + step
    assert calls["umic_cache_attention_bf16"] == calls["umic_qk_rmsnorm_rope_kv_append_bf16"] == 12
    assert integrate.unfuse_mlps(m) == 2
    assert not hasattr(m.layers[0].self_attn, "_umic_cache_attention")


def test_a_step_that_is_not_causal(calls):
    """An action expert's tokens see the prefix and each other; a causal prompt and a masked call
    stay on SDPA."""
    from transformers.cache_utils import DynamicCache

    m, _ = text_model(kv_heads=4)
    integrate.fuse_cache_attention(m)
    attn = m.layers[0].self_attn
    g = torch.Generator().manual_seed(6)
    prefix = DynamicCache()
    k0, v0 = (torch.randn(1, 4, 50, 128, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    prefix.update(k0, v0, 0)
    x = torch.randn(1, 12, 256, generator=g).to(torch.bfloat16).to(DEV)
    rot = m.rotary_emb(x, torch.arange(50, 62, device=DEV).expand(3, 1, 12))
    with torch.no_grad():
        outs = []
        for on, causal in ((True, False), (False, False), (True, True)):
            attn._umic_cache_attention, attn.is_causal = on, causal
            c = InplaceKVCache.from_dynamic(prefix, extra_tokens=16)
            before = calls["umic_cache_attention_bf16"]
            if not on:  # every key is seen: a mask of all ones
                mask = torch.ones(1, 1, 12, 62, dtype=torch.bool, device=DEV)
                attn._umic_cache_attention = True
            else:
                mask = None
            outs.append(attn(x, rot, mask, past_key_values=c)[0])
            assert (calls["umic_cache_attention_bf16"] > before) == (on and not causal)
            assert c.get_seq_length() == 62
    assert rel_err(outs[0], outs[1]) <= TOL


def test_decode_graphs_with_cache_attention(calls):
    """generate() through the per-length graphs, each with the kernel in it: the eager tokens."""
    from test_gpu_decode_graph import generate, small_vlm
    from torch.nn.attention import SDPBackend, sdpa_kernel

    m = small_vlm()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 512, (1, n), generator=g).to(DEV) for n in (24, 24, 24, 17)]
    with torch.no_grad(), sdpa_kernel([SDPBackend.FLASH_ATTENTION,
                                       SDPBackend.EFFICIENT_ATTENTION]):
        want = [generate(m, p) for p in prompts]
        lm = m.model.language_model
        assert integrate.fuse_kv_rope(lm) == integrate.fuse_cache_attention(lm) == 2
        runner = DecodeGraphRunner(m, max_new_tokens=16)
        for p, (tokens, scores) in zip(prompts, want):
            got, gs = generate(m, p)
            assert rel_err(gs[0], scores[0]) <= TOL
            # greedy tokens part where two scores tie within the tolerance
            same = (got == tokens).all().item()
            assert same or (scores.topk(2).values.diff().abs().min()
                            <= 2 * TOL * scores.abs().max()), (got, tokens)
    assert runner.replays > 0 and calls["umic_cache_attention_bf16"] > 0
