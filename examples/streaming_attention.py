"""Series that keep growing: time attention of one encoder layer over a 4-bit K/V cache.

Each series' past patches have their keys and values appended to a paged cache once; every new patch then costs one
token: its projections, one append, one attention over everything cached.  The layer's weights are the model's; attention
is causal, so that one layer's cached keys do not depend on later patches (the model's own forward lets patches see later
ones, and recomputes them).

The series stand in for a stream: all patches are embedded at the start, the later ones too.  The model's embedding scales
a series by its mean and deviation and counts its time encoding from the end, and both move with every new value.  A stream
has to fix them (the past's, say) or to encode and append anew; with those that change under it, what is cached goes out of
date.  Prints what the cache takes next to bf16 and how far its attention is from dense attention over
unquantised keys and values.

    python examples/streaming_attention.py [--series 16] [--context 4096] [--steps 32]
"""

from __future__ import annotations

import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from cutechronos_b200 import CuteChronos2Config, CuteChronos2Model, kernels  # noqa: E402
from cutechronos_b200.kvcache import rope_rows  # noqa: E402
from cutechronos_b200.workloads import seeded_init_, series_cfg1  # noqa: E402


def embed(model: CuteChronos2Model, context: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(series, length) values -> patch embeddings (series, patches, d_model) and which patches have data."""
    cfg, e = model.config, model.input_patch_embedding
    patches, mask, _, _ = kernels.fused_preprocess(context, cfg.input_patch_size, cfg.context_length, cfg.use_arcsinh,
                                                   time_encoding_scale=cfg.time_encoding_scale, dtype=torch.bfloat16)
    hidden = kernels.linear(patches, e.hidden_layer.weight, e.hidden_layer.bias, relu=True)
    skip = kernels.linear(patches, e.residual_layer.weight, e.residual_layer.bias)
    return kernels.linear(hidden, e.output_layer.weight, e.output_layer.bias, residual=skip.view(-1, cfg.d_model)), mask > 0


def project(model: CuteChronos2Model, layer: int, x: torch.Tensor):
    """Tokens (n, d_model) -> q, k, v (n, heads, 64) of the layer's time attention, not yet rotated."""
    att, cfg = model.blocks[layer].time_attn, model.config
    h = kernels.rms_layernorm(x, att.layer_norm_weight, cfg.layer_norm_epsilon)
    return [kernels.linear(h, p.weight).view(-1, cfg.num_heads, 64) for p in (att.q, att.k, att.v)]


def dense(q, k, v, mask, theta: float):
    """Causal attention in fp32 over unquantised keys and values: q, k, v (series, tokens, heads, 64)."""
    cs = rope_rows(q.shape[1], theta, q.device)[None, :, None]
    turn = lambda x: torch.cat([x[..., :32] * cs[..., 0] - x[..., 32:] * cs[..., 1],  # noqa: E731
                                x[..., 32:] * cs[..., 0] + x[..., :32] * cs[..., 1]], -1)
    s = torch.einsum("bihd,bjhd->bhij", turn(q.float()), turn(k.float()))
    n = q.shape[1]
    see = torch.ones(n, n, dtype=torch.bool, device=q.device).tril() & mask[:, None, None, :]
    p = s.masked_fill(~see, -torch.inf).softmax(-1)
    return torch.einsum("bhij,bjhd->bihd", torch.where(see, p, 0.0), v.float())


@torch.inference_mode()
def main(series: int = 16, context: int = 4096, steps: int = 32, page_size: int = 64, layer: int = 0,
         config: CuteChronos2Config | None = None) -> dict:
    model = seeded_init_(CuteChronos2Model(config or CuteChronos2Config(num_layers=1)), seed=0)
    model = model.to("cuda", torch.bfloat16).eval()
    cfg, dev = model.config, "cuda"
    x, mask = embed(model, series_cfg1(series, context, 0).to(dev))
    tokens = x.shape[1]
    past = tokens - steps
    assert past > 0, "more steps than patches"
    q, k, v = (t.view(series, tokens, cfg.num_heads, 64) for t in project(model, layer, x.reshape(-1, cfg.d_model)))

    # a page table row for each series; a server would hand pages out as the series grow
    width = -(-tokens // page_size)
    cache = model.kv4_cache(series * width, layer=layer, page_size=page_size, max_positions=tokens)
    table = torch.randperm(series * width, device=dev).view(series, width).int()
    ids = torch.arange(series, device=dev, dtype=torch.int32)

    # the past: one append, one attention
    seq, pos = ids.repeat_interleave(past), torch.arange(past, device=dev, dtype=torch.int32).repeat(series)
    cache.append(k[:, :past].reshape(-1, cfg.num_heads, 64), v[:, :past].reshape(-1, cfg.num_heads, 64), seq, pos, table,
                 token_mask=mask[:, :past].reshape(-1))
    lens = torch.full((series,), past, dtype=torch.int32, device=dev)
    out = [cache.attention(q[:, :past].reshape(-1, cfg.num_heads, 64), lens, table, max_len=tokens,
                           rotate_q=True).view(series, past, cfg.num_heads, 64)]
    # new patches, one token for each series at a time
    for i in range(past, tokens):
        cache.append(k[:, i], v[:, i], ids, lens, table, token_mask=mask[:, i])
        lens += 1
        out.append(cache.attention(q[:, i], lens, table, max_len=tokens, rotate_q=True)[:, None])
    cache.check()
    out = torch.cat(out, 1)
    ref = dense(q, k, v, mask, cfg.rope_theta)
    update = kernels.linear(out.reshape(-1, cfg.num_heads * 64), model.blocks[layer].time_attn.o.weight)
    err = ((out.float() - ref).norm() / ref.norm()).item()
    dense_bytes = 2 * series * tokens * cfg.num_heads * 64 * 2
    print(f"{series} series x {tokens} patches x {cfg.num_heads} heads: cache {cache.pages.numel() / 2**20:.2f} MiB "
          f"(bf16 {dense_bytes / 2**20:.2f}), attention off by {err:.3f} of its norm")
    return dict(error=err, ratio=dense_bytes / cache.pages.numel(), output=out, reference=ref, update=update)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    for name, default in (("series", 16), ("context", 4096), ("steps", 32), ("page-size", 64)):
        ap.add_argument(f"--{name}", type=int, default=default)
    main(**{k.replace("-", "_"): v for k, v in vars(ap.parse_args()).items()})
