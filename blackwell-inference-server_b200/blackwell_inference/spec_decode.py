"""Speculative decoding of a registry's model over a paged int8 KV cache.

``TreeSpeculativeDecoder`` runs a Hugging Face decoder whose projections a ``MultiDeltaLoRAModel`` holds as
W8A16 copies (Llama- and Qwen3-style layers) without the model's own cache and attention: one forward pass
takes the nodes of a tree of drafted tokens, and a layer is

    rmsnorm -> int8_gemm_grouped (q, k, v) -> rotary_kv_write_int8 -> tree_attention_int8 -> int8_gemm
    -> residual -> rmsnorm -> int8_gemm_swiglu -> int8_gemm -> residual.

The drafts come from a lookup in the tokens so far (the idea of the reference's n-gram proposer,
``src/blackwell_inference/spec/ngram.py:25-57``, which proposes one chain): the continuations of the last
tokens' earlier occurrences, merged into a tree.  ``verify_tree`` accepts them so that the tokens are
distributed as the model alone would draw them, ``kv_move_int8`` moves the accepted nodes' cache rows to
their final slots, and the last token is the next tree's root.

    mdl = MultiDeltaLoRAModel(model, device="cuda")
    dec = TreeSpeculativeDecoder(mdl, batch=1, max_len=4096)
    new = dec.generate(ids, max_new_tokens=64, adapter="a")
"""
from __future__ import annotations

import torch

from .lora.delta_multi import MultiDeltaLoRAModel, W8A16Linear


def lookup_tree(tokens: list[int], nodes: int, branches: int = 4, ngram: int = 3) -> tuple[list[int], list[int]]:
    """Drafted tokens and parents of a tree of at most ``nodes`` nodes whose root is ``tokens[-1]``.

    The latest ``branches`` earlier occurrences of the last ``ngram`` tokens (or of fewer, where they have
    none) give one continuation each; common beginnings are one node.  A longer match goes first, and a
    later one before an earlier.  A scan of the text on the host, one to three ms for 4000 tokens without a match."""
    out, parents = [tokens[-1]], [-1]
    if nodes <= 1:
        return out, parents
    children: dict[tuple[int, int], int] = {}
    found = 0
    for n in range(min(ngram, len(tokens) - 1), 0, -1):
        tail = tokens[-n:]
        for at in range(len(tokens) - n - 1, -1, -1):
            if tokens[at:at + n] != tail:
                continue
            cur = 0
            for tok in tokens[at + n:at + n + (nodes - 1) // branches + 1]:
                nxt = children.get((cur, tok))
                if nxt is None:
                    if len(out) == nodes:
                        break
                    nxt = children[(cur, tok)] = len(out)
                    out.append(tok)
                    parents.append(cur)
                cur = nxt
            found += 1
            if found == branches or len(out) == nodes:
                return out, parents
        if found:
            break
    return out, parents


def _fusable(projections) -> bool:
    """int8 copies and nothing else to add: one launch can take them together."""
    return all(isinstance(p, W8A16Linear) and p.bias is None for p in projections)


# Models whose layers are what `forward` computes.  Others name their modules alike and scale embeddings, residuals or
# logits, interleave the rotated pairs, offset the norms' weights or leave layers without positions.
MODEL_TYPES = ("llama", "mistral", "qwen2", "qwen3")


def _check_attention(cfg, positions: int) -> None:
    """Every layer attends to all of its sequence, or to a window that no position leaves."""
    window = getattr(cfg, "sliding_window", None)
    if not getattr(cfg, "use_sliding_window", True):
        window = None
    kinds = set(getattr(cfg, "layer_types", None) or (["full_attention"] if window is None else ["sliding_attention"]))
    for kind in sorted(kinds - {"full_attention", "sliding_attention"}):
        raise RuntimeError(f"layers of {kind} are not supported")
    if "sliding_attention" in kinds and (window is None or window < positions):
        raise RuntimeError(f"a window of {window} tokens is shorter than max_len and the nodes of a step, {positions}: "
                           "not supported")


def _rope(cfg) -> dict:
    """The model's rotation as ``rotary_plan`` takes it, with its ``rope_theta``: ``rope_parameters``, or the attributes
    ``rope_scaling`` and ``rope_theta`` of older configurations."""
    rope = dict(getattr(cfg, "rope_parameters", None) or getattr(cfg, "rope_scaling", None) or {})
    rope.setdefault("rope_theta", getattr(cfg, "rope_theta", 10000.0))
    for part in (rope.get("partial_rotary_factor"), getattr(cfg, "partial_rotary_factor", None)):
        if part is not None and part != 1:
            raise RuntimeError(f"partial_rotary_factor {part}: heads that turn in part are not supported")
    return rope


class TreeSpeculativeDecoder:
    """Decodes ``batch`` sequences of at most ``max_len`` tokens, ``nodes`` tree nodes a step (1: plain decoding).

    Takes models of ``MODEL_TYPES``.  Attention windows shorter than ``max_len + nodes``, heads that turn in part and
    rotations that ``rotary_frequencies`` does not know are refused."""

    def __init__(self, model: MultiDeltaLoRAModel, batch: int, max_len: int, nodes: int = 16, page: int = 64):
        from blackwell_ops.decode import MAX_NODES, KVCacheInt8, rotary_plan

        if not model.quantize:
            raise RuntimeError("the registry must hold int8 copies (quantize=True)")
        if not 1 <= nodes <= MAX_NODES:
            raise RuntimeError(f"1 to {MAX_NODES} nodes a step")
        self.model, self.batch, self.nodes = model, batch, nodes
        self.max_len = max_len
        cfg = model.base.config
        if cfg.model_type not in MODEL_TYPES:
            raise RuntimeError(f"models of type {cfg.model_type!r} are not supported, only {', '.join(MODEL_TYPES)}")
        _check_attention(cfg, max_len + nodes)
        rope = _rope(cfg)
        self.head_dim = getattr(cfg, "head_dim", None) or cfg.hidden_size // cfg.num_attention_heads
        self.heads, self.kv_heads = cfg.num_attention_heads, cfg.num_key_value_heads
        self.swiglu = getattr(cfg, "hidden_act", None) in ("silu", "swish")  # the fused gate and up product's
        self.layers = model.base.model.layers
        self.dev = next(model.base.parameters()).device
        self.plan = rotary_plan(self.head_dim, float(rope["rope_theta"]), rope, device=self.dev)
        per = -(-(max_len + nodes) // page)
        self.cache = KVCacheInt8.empty(batch * per, self.kv_heads, page, self.head_dim, len(self.layers), self.dev)
        self._layer_cache = [self.cache.layer(i) for i in range(len(self.layers))]
        self.table = torch.arange(batch * per, dtype=torch.int32, device=self.dev).view(batch, per)
        self.ctx = torch.zeros(batch, dtype=torch.int32, device=self.dev)

    def reset(self) -> None:
        self.ctx.zero_()

    @torch.no_grad()
    def forward(self, tokens: torch.Tensor, parents: torch.Tensor | None = None, logits: bool = True) -> torch.Tensor | None:
        """Logits [B, T, V] after each node of a tree ``tokens``, ``parents`` [B, T] (None: a chain) that follows
        the committed tokens.  The nodes' keys and values go to slots ``ctx`` on; nothing is committed."""
        from blackwell_ops.cuda import rmsnorm
        from blackwell_ops.decode import rotary_kv_write_int8, tree_attention_int8, tree_positions
        from blackwell_ops.kernels.int8_gemm import int8_gemm_grouped

        b, t = tokens.shape
        mask = None
        if parents is None:
            pos = self.ctx[:, None] + torch.arange(t, dtype=torch.int32, device=self.dev)
        else:
            mask, pos = tree_positions(parents, self.ctx)
        x = self.model.base.model.embed_tokens(tokens).reshape(b * t, -1)
        for layer, cache in zip(self.layers, self._layer_cache):
            att, mlp = layer.self_attn, layer.mlp
            y = rmsnorm(x, layer.input_layernorm.weight, layer.input_layernorm.variance_epsilon)
            proj = (att.q_proj, att.k_proj, att.v_proj)
            if _fusable(proj):
                q, k, v = int8_gemm_grouped(y, [p.copies[p.active] for p in proj])
            else:
                q, k, v = (p(y) for p in proj)
            q, k = self._head_norm(q, getattr(att, "q_norm", None)), self._head_norm(k, getattr(att, "k_norm", None))
            shape = (b, t, -1, self.head_dim)
            q = rotary_kv_write_int8(q.view(shape), k.view(shape), v.view(shape), pos, self.plan, cache, self.table, self.ctx)
            o = tree_attention_int8(q, cache, self.table, self.ctx, mask, softmax_scale=att.scaling)
            x = x + att.o_proj(o.view(b * t, -1))
            y = rmsnorm(x, layer.post_attention_layernorm.weight, layer.post_attention_layernorm.variance_epsilon)
            x = x + self._mlp(mlp, y)
        if not logits:
            return None
        norm = self.model.base.model.norm
        return self.model.base.lm_head(rmsnorm(x, norm.weight, norm.variance_epsilon)).view(b, t, -1)

    def _mlp(self, mlp, y: torch.Tensor) -> torch.Tensor:
        from blackwell_ops.kernels.int8_gemm import int8_gemm, int8_gemm_swiglu

        proj = (mlp.gate_proj, mlp.up_proj, mlp.down_proj)
        if not self.swiglu or not _fusable(proj):
            return mlp.down_proj(mlp.act_fn(mlp.gate_proj(y)) * mlp.up_proj(y))
        (wg, sg), (wu, su), (wd, sd) = (p.copies[p.active] for p in proj)
        return int8_gemm(int8_gemm_swiglu(y, wg, sg, wu, su), wd, sd)

    def _head_norm(self, x: torch.Tensor, norm) -> torch.Tensor:
        """Qwen3 normalises each head of q and k."""
        from blackwell_ops.cuda import rmsnorm

        if norm is None:
            return x
        return rmsnorm(x.view(-1, self.head_dim), norm.weight, norm.variance_epsilon).view(x.shape)

    def commit(self, path: torch.Tensor, taken: torch.Tensor) -> None:
        """Keep the root and the accepted nodes ``path[b, :taken[b]]`` of the last forward pass."""
        from blackwell_ops.decode import kv_move_int8

        kv_move_int8(self.cache, self.table, self.ctx, path, taken)
        self.ctx += taken + 1

    def prefill(self, tokens: torch.Tensor) -> None:
        """Commit ``tokens`` [B, L], in chains of at most 64."""
        for at in range(0, tokens.shape[1], 64):
            part = tokens[:, at:at + 64]
            self.forward(part, logits=False)
            self.ctx += part.shape[1]

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, max_new_tokens: int, adapter: str | None = None, temperature: float = 0.0,
                 generator: torch.Generator | None = None) -> torch.Tensor:
        """The new tokens [B, max_new_tokens] after the prompts ``ids`` [B, L]; ``temperature`` 0 is greedy."""
        from blackwell_ops.decode import verify_tree

        b, length = ids.shape
        if b != self.batch or length < 1:
            raise RuntimeError(f"ids must be [{self.batch}, L] with L >= 1")
        if max_new_tokens < 0:
            raise RuntimeError("max_new_tokens must not be negative")
        if length + max_new_tokens > self.max_len:
            raise RuntimeError(f"at most max_len = {self.max_len} tokens a sequence")
        self.model.set_adapter(adapter)
        self.reset()
        ids = ids.to(self.dev)
        self.prefill(ids[:, :-1])
        seen = ids.tolist()
        while min(len(s) for s in seen) < length + max_new_tokens:
            # (a sequence that has its tokens goes on with its root alone, whose place is kept)
            trees = [lookup_tree(s, min(self.nodes, max(1, length + max_new_tokens - len(s)))) for s in seen]
            t = max(len(tok) for tok, _ in trees)
            tokens = torch.tensor([tok + [0] * (t - len(tok)) for tok, _ in trees], device=self.dev)
            parents = torch.tensor([p + [-1] * (t - len(p)) for _, p in trees], dtype=torch.int32, device=self.dev)
            logits = self.forward(tokens, parents).float()
            if temperature > 0:
                probs = torch.softmax(logits / temperature, -1)
            else:
                probs = torch.zeros_like(logits).scatter_(-1, logits.argmax(-1, keepdim=True), 1.0)
            u = torch.rand((b, t), generator=generator, device=self.dev)
            e = torch.empty((b, probs.shape[-1]), device=self.dev).exponential_(generator=generator)
            n, path, out = verify_tree(probs, tokens, parents, u, e)
            full = torch.tensor([len(s) >= length + max_new_tokens for s in seen], device=self.dev)
            before = self.ctx.clone()
            self.commit(path, n)
            self.ctx = torch.where(full, before, self.ctx)
            for s, k, new in zip(seen, n.tolist(), out.tolist()):
                if len(s) < length + max_new_tokens:
                    s += new[:k + 1]
        return torch.tensor([s[length:length + max_new_tokens] for s in seen], dtype=torch.int64, device=self.dev)
