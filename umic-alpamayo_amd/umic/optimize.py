"""One-call UMIC application: ``umic.apply(model)``.

Same API as the reference (src/umic/optimize.py): a ``UmicConfig`` of flags
and ``apply(model, config) -> report`` that patches every configured fusion
in place and returns per-fusion match counts (0 = motif not found, that
fusion is a no-op).  Matching is structural, so the call works on any model
that keeps the motifs (gate/up/down SiLU MLP, pre-norm decoder layer,
RMSNorm / LayerNorm, transformers qwen3_vl RoPE).

This runtime implements the kernel fusions of the hot path on gfx950:
P5 MLP, q/o projections, RMSNorm, add+RMSNorm, LayerNorm, the ViT
add+LayerNorm pipeline and text / vision RoPE, plus the in-place KV cache
(flow_cache, decode_cache) with the text RoPE fused into its append and the
per-KV-length decode graphs (decode_graph).  The reference's approximate flow
step skipping (adaptive_flow) and the ViT patch-embed / packed-attention /
bf16-residual rewrites inside vision_fusion are not part of it: their flags
are accepted for API compatibility and reported as not applied.
"""

from __future__ import annotations

import dataclasses
import logging

from torch import nn

logger = logging.getLogger(__name__)


@dataclasses.dataclass
class UmicConfig:
    """Which optimizations to apply (defaults: the reference's adopted set).

    Attributes:
        mlp_fusion: P5 gate_silu_mul fusion on the LM trunk MLPs.
        linear_fusion: q/o projections on the fused MFMA linear.
        norm_fusion: fused RMSNorm on the LM trunk (and on the flow expert
            when flow_cache is set, as every expert fusion).
        add_rmsnorm_fusion: attention-residual add folded into the
            post-attention RMSNorm (LM and expert decoder layers).
        text_rope_fusion: fused text RoPE (transformers qwen3_vl global).
        vision_fusion: ViT fused LayerNorm, vision RoPE and the
            add+LayerNorm pipeline (grid_thw constants cache).
        gelu_mlp_fusion: with vision_fusion, the ViT blocks' fc1 + GELU on
            the fused linear with a GELU epilogue (erf or tanh form, as the
            module computes).  The reference provides fuse_gelu_mlps but
            leaves it out of its adopted set; on MI355X it is a gain.
        flow_cache: in-place KV cache for the flow expert's
            append-then-crop loop.
        decode_cache: in-place KV cache for autoregressive decode (used
            when decode_graph is off; the graph runner owns its cache).
        decode_graph: per-KV-length decode HIP graphs, persistent across
            inferences (umic.graph.DecodeGraphRunner).
        adaptive_flow: accepted for compatibility; not implemented
            (reported False).
        max_new_tokens: decode-graph KV headroom (>= generate() budget).
        cache_attention: with text_rope_fusion, single tokens and steps that
            are not causal attend over the in-place cache with the library's
            kernel instead of SDPA (no reference counterpart; off, as SDPA's
            results are kept).
    With text_rope_fusion, attention calls that append to an in-place
    cache rotate q/k and write the cache in one launch.
    """

    mlp_fusion: bool = True
    linear_fusion: bool = True
    norm_fusion: bool = True
    add_rmsnorm_fusion: bool = True
    text_rope_fusion: bool = True
    vision_fusion: bool = True
    gelu_mlp_fusion: bool = True
    flow_cache: bool = True
    decode_cache: bool = True
    decode_graph: bool = True
    adaptive_flow: bool = False
    max_new_tokens: int = 96
    cache_attention: bool = False


def find_lm_module(model: nn.Module) -> nn.Module | None:
    """Locate the LM trunk under model.vlm (duck-typed, version-agnostic).

    The reference's lookup (vlm.language_model or vlm.model, holding
    ``layers`` directly or one ``.model`` down), plus transformers >= 5's
    layout, where Qwen3VLForConditionalGeneration no longer exposes
    ``language_model`` and the trunk is vlm.model.language_model."""
    vlm = getattr(model, "vlm", None)
    if vlm is None:
        return None
    for attr in ("language_model", "model"):
        cand = getattr(vlm, attr, None)
        if cand is None:
            continue
        if hasattr(cand, "layers"):
            return cand
        sub = getattr(cand, "model", None)
        if sub is not None and hasattr(sub, "layers"):
            return cand
        inner = getattr(cand, "language_model", None)
        if inner is not None and hasattr(inner, "layers"):
            return inner
    return None


def find_visual_module(model: nn.Module) -> nn.Module | None:
    """The vision encoder: model.vlm.visual, or model.vlm.model.visual
    (transformers >= 5's Qwen3VLForConditionalGeneration)."""
    vlm = getattr(model, "vlm", None)
    visual = getattr(vlm, "visual", None)
    if visual is None:
        visual = getattr(getattr(vlm, "model", None), "visual", None)
    return visual


def _hook(fn):
    """A step whose action installs a hook and reports True."""
    def run(module, cfg):
        fn(module, cfg)
        return True
    return run


def _plan(integrate):
    """The fusions in application order, one row each:
    (condition on the config, module scope, report key, action(module, cfg)).

    Scopes: "lm" the LM trunk, "visual" the vision encoder, "expert" the flow
    expert, "vlm" the VLM, None the model itself (process-wide patches).  The
    report keys and their conditions are the reference's contract
    (src/umic/optimize.py:92-168), plus this runtime's additions:
    lm_kv_rope_fused / expert_kv_rope_fused (text RoPE fused into the
    in-place cache append), lm_cache_attention / expert_cache_attention and
    ve_gelu_mlp_fused.  The reference's ViT
    patch-embed, packed-attention and bf16-residual rewrites are not part of
    this runtime, so their keys never appear.
    """
    from umic.graph import fuse_decode_graph

    def count(name):
        fn = getattr(integrate, name)
        return lambda module, cfg: fn(module)

    def glob(name):
        fn = getattr(integrate, name)
        return lambda module, cfg: fn()

    def skipped_adaptive_flow(module, cfg):
        logger.info("umic.apply: adaptive_flow is not implemented by this runtime; skipped")
        return False

    return (
        (lambda c: c.mlp_fusion, "lm", "lm_mlp_fused", count("fuse_mlps")),
        (lambda c: c.linear_fusion, "lm", "lm_linear_fused", count("fuse_linears")),
        (lambda c: c.norm_fusion, "lm", "lm_rmsnorm_fused", count("fuse_rmsnorms")),
        (lambda c: c.add_rmsnorm_fusion, "lm", "lm_add_rmsnorm_fused",
         count("fuse_add_rmsnorm")),
        (lambda c: c.text_rope_fusion, None, "text_rope_fused", glob("fuse_text_rope")),
        (lambda c: c.text_rope_fusion, "lm", "lm_kv_rope_fused", count("fuse_kv_rope")),
        (lambda c: c.vision_fusion, "visual", "ve_layernorm_fused", count("fuse_layernorms")),
        (lambda c: c.vision_fusion, "visual", "ve_rope_fused", glob("fuse_vision_rope")),
        (lambda c: c.vision_fusion, "visual", "ve_pipeline_fused",
         count("fuse_vision_encoder_pipeline")),
        (lambda c: c.vision_fusion and c.gelu_mlp_fusion, "visual", "ve_gelu_mlp_fused",
         count("fuse_gelu_mlps")),
        (lambda c: c.flow_cache, "expert", "flow_cache_hook",
         _hook(lambda m, c: integrate.fuse_repeat_cache(m))),
        (lambda c: c.flow_cache and c.norm_fusion, "expert", "expert_rmsnorm_fused",
         count("fuse_rmsnorms")),
        (lambda c: c.flow_cache and c.add_rmsnorm_fusion, "expert", "expert_add_rmsnorm_fused",
         count("fuse_add_rmsnorm")),
        (lambda c: c.flow_cache and c.text_rope_fusion, "expert", "expert_kv_rope_fused",
         count("fuse_kv_rope")),
        (lambda c: c.cache_attention and c.text_rope_fusion, "lm", "lm_cache_attention",
         count("fuse_cache_attention")),
        (lambda c: c.cache_attention and c.flow_cache and c.text_rope_fusion, "expert",
         "expert_cache_attention", count("fuse_cache_attention")),
        (lambda c: c.decode_graph, "vlm", "decode_graph",
         _hook(lambda m, c: fuse_decode_graph(m, max_new_tokens=c.max_new_tokens))),
        (lambda c: c.decode_cache and not c.decode_graph, "vlm", "decode_cache_hook",
         _hook(lambda m, c: integrate.fuse_repeat_cache(m, extra_tokens_hint=128))),
        (lambda c: c.adaptive_flow, None, "adaptive_flow", skipped_adaptive_flow),
    )


def apply(model: nn.Module, config: UmicConfig | None = None) -> dict:
    """Patch all configured UMIC fusions into `model`, in place.

    Args:
        model: An Alpamayo-family model (``model.vlm`` with its language model
            and ``visual`` encoder, optional ``model.expert``); weights untouched.
        config: Optional UmicConfig; defaults to the full adopted set.

    Returns:
        Report dict: per-fusion match counts (0 = motif not found) or True for
        installed hooks; a step whose module is absent is left out.
    """
    from umic import integrate

    cfg = config or UmicConfig()
    scopes = {"lm": find_lm_module(model), "visual": find_visual_module(model),
              "expert": getattr(model, "expert", None), "vlm": getattr(model, "vlm", None),
              None: model}
    if scopes["lm"] is None:
        logger.warning("umic.apply: no LM trunk found under model.vlm -- LM fusions skipped")
    report: dict[str, object] = {}
    for wanted, scope, key, run in _plan(integrate):
        module = scopes[scope]
        if wanted(cfg) and module is not None:
            report[key] = run(module, cfg)
    logger.info("umic.apply report: %s", report)
    return report
