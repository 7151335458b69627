"""The plain implementation with its layers' products in 8 bits: weights and tokens rounded as the 8-bit operators
define it (a row's largest magnitude is 127 steps), everything else as in ``plain_qwen3``."""
import torch

import plain_qwen3 as plain


def rows(t):
    """Each row as its 8-bit integers stand for it."""
    most = t.abs().amax(-1, keepdim=True).clamp_min(127 * 2.0 ** -126)
    return torch.round(t * (127 / most)) * (most / 127)


class _Attention:
    """What ``plain.attention`` rounds on its way, in order: q, k, v, rotated q and k, each head's weights, and at last
    the output, whose rows go into the O product in 8 bits."""

    def __init__(self, nq, rnd):
        self.left, self.rnd = 5 + nq, rnd

    def __call__(self, t):
        self.left -= 1
        return rows(self.rnd(t)) if self.left < 0 else self.rnd(t)


def forward(cfg, w, tokens, rnd=lambda t: t):
    """Logits [T, vocab]; ``rnd`` imitates where a 16-bit engine stores activations (not the normed rows, which go
    into 8 bits at once)."""
    w = {k: v.to(torch.float32) for k, v in w.items()}
    nq = cfg["num_attention_heads"]
    nkv, hd, eps = cfg.get("num_key_value_heads", nq), cfg.get("head_dim") or cfg["hidden_size"] // nq, cfg["rms_norm_eps"]
    freqs, mscale = plain.rope_frequencies(hd, cfg["rope_theta"], plain._scaling(cfg))
    x = w["model.embed_tokens.weight"][torch.as_tensor(tokens, dtype=torch.long)]
    for l in range(cfg["num_hidden_layers"]):
        p = f"model.layers.{l}."
        m = {k: rows(w[f"{p}{part}.{k}_proj.weight"]) for part, names in (("self_attn", "qkvo"), ("mlp", ("gate", "up", "down")))
             for k in names}
        n = rows(plain.rmsnorm(x, w[p + "input_layernorm.weight"], eps))
        x = x + plain.attention(n, m["q"], m["k"], m["v"], m["o"], w[p + "self_attn.q_norm.weight"], w[p + "self_attn.k_norm.weight"],
                                nq, nkv, hd, eps, freqs, mscale, hd, rnd=_Attention(nq, rnd))
        n = rows(plain.rmsnorm(x, w[p + "post_attention_layernorm.weight"], eps))
        x = x + plain.swiglu(n, m["gate"], m["up"], m["down"], lambda t: rows(rnd(t)))
    x = rnd(plain.rmsnorm(x, w["model.norm.weight"], eps))
    head = w["lm_head.weight"] if not cfg.get("tie_word_embeddings", False) else w["model.embed_tokens.weight"]
    return x @ head.T
