"""GPU: generate() through the per-length decode graphs with fuse_cache_attention's kernel in them,
every step's scores against the unpatched model's.

Greedy decoding is followed up to the first step whose tokens differ, that step included: its inputs
are still alike, and scores within the tolerance can only part there where two of them tie.  The
tolerance is that of this package's layer tests: both sides round to bf16 after every operation, in
other places."""

from __future__ import annotations

import copy

import pytest
import torch

from helpers import rel_err
from test_gpu_decode_graph import NEW, generate, small_vlm
from test_gpu_paged_cache import TOL, calls  # noqa: F401 (a fixture)
from umic import integrate
from umic.graph import DecodeGraphRunner

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore::FutureWarning"),
              pytest.mark.filterwarnings("ignore::UserWarning")]
DEV = "cuda"


def steps_alike(got, want):
    """Steps whose inputs are alike: up to the first whose tokens differ."""
    tokens, scores = got
    n = 0
    for a, b in zip(scores.argmax(-1).flatten(), want[1].argmax(-1).flatten()):
        n += 1
        if a != b:
            break
    held = tokens.shape[1] - len(scores)
    assert torch.equal(tokens[:, :held + n - 1], want[0][:, :held + n - 1])
    return n


def test_every_step_of_the_graphs_is_the_eager_one(calls):  # noqa: F811
    from torch.nn.attention import SDPBackend, sdpa_kernel

    m = small_vlm()
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, 512, (1, n), generator=g).to(DEV) for n in (24, 24, 24, 17, 130)]
    with torch.no_grad(), sdpa_kernel([SDPBackend.FLASH_ATTENTION,
                                       SDPBackend.EFFICIENT_ATTENTION]):
        want = [generate(m, p) for p in prompts]
        # the attention weighs in these scores many times what they may be off
        deaf = copy.deepcopy(m)
        for layer in deaf.model.language_model.layers:
            layer.self_attn.o_proj.weight.zero_()
        for p in prompts:
            assert rel_err(deaf(input_ids=p).logits[0, -1:], m(input_ids=p).logits[0, -1:]) > 10 * TOL
        lm = m.model.language_model
        assert integrate.fuse_kv_rope(lm) == integrate.fuse_cache_attention(lm) == 2
        runner = DecodeGraphRunner(m, max_new_tokens=16)
        compared = []
        for p, w in zip(prompts, want):
            before = calls["umic_cache_attention_bf16"], runner.replays
            got = generate(m, p)
            n = steps_alike(got, w)
            compared.append(n - 1)  # the first step is the prompt's, not the kernel's
            for i in range(n):
                assert rel_err(got[1][i], w[1][i]) <= TOL, (p.shape, i)
            assert calls["umic_cache_attention_bf16"] > before[0] or runner.replays > before[1]
    # every prompt has steps of the kernel that were compared, and most of all steps were
    print("steps compared", compared)
    assert min(compared) >= 1 and sum(compared) >= len(prompts) * (NEW - 1) // 3
    assert runner.replays > 0 and calls["umic_cache_attention_bf16"] > 0
