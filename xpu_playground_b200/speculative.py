"""Speculative decoding over the paged cache: the serving operators together.

A Qwen3 of any preset, with the engine's seeded synthetic weights, serves several
prompts at once: the prompts go through each layer packed
(``kernels.prompt_attention``) and their keys and values into the cache's pages
(``KvCache.extend`` / ``write``); each prompt is forked into ``samples`` sequences
that begin with its most likely tokens (``KvCache.fork``); every step then verifies
a tree of drafted tokens per sequence in one forward pass
(``kernels.tree_attention``), appends the accepted ones (``KvCache.append``), and
frees sequences that are done (``KvCache.trim``, ``KvCache.compact``). Drafts come
from the sequence's own text: what followed the last occurrences of its newest
token. With ``width`` 0 a tree is one node and the loop is plain greedy decoding;
drafts change how many steps it takes, not the tokens (up to logits that differ
by no more than their rounding). With a ``Sampling`` every token is drawn
(``kernels.sample``) instead, from a random number of its own sequence and position, so
that drafts do not change it either: a drafted token stands where it is the one drawn. The
seed and the requests before decide the numbers: the same prompt again is drawn anew.

With ``eight_bits`` the projections are held and multiplied in 8 bits: the residual's
addition and the norm (``kernels.fp8_rms_norm``), the attention's output
(``kernels.fp8_quantize``) and the gated activation (``kernels.fp8_silu_multiply``) leave
as 8-bit rows, which enter ``kernels.fp8_gemm``.

    python -m xpu_playground_b200.speculative --preset tiny --prompts 3 --new-tokens 48
    python -m xpu_playground_b200.speculative --eight-bits --temperature 0.7 --top-k 20 --top-p 0.95
"""

from __future__ import annotations

import argparse
import json
import time
from dataclasses import dataclass, field

import torch

from . import _lib, kernels
from .fp8 import Fp8Weight
from .kv_cache import KvCache
from .qwen3_config import HEAD_DIM, PRESETS, WEIGHT_STD, Qwen3Shape


def synthetic_weights(shape: Qwen3Shape, seed: int, std: float = WEIGHT_STD) -> dict[str, torch.Tensor]:
    """The tensors that xpu_qwen3_init_synthetic draws, bit for bit."""
    weights = {}
    for name in shape.tensor_names():
        size = shape.shape_of(name)
        if shape.is_norm(name):
            weights[name] = torch.ones(size, dtype=torch.bfloat16, device="cuda")
            continue
        t = torch.empty(size, dtype=torch.bfloat16, device="cuda")
        _lib.call("xpu_fill_normal_bf16", t.data_ptr(), t.numel(), seed, shape.tensor_tag(name), std, kernels._stream())
        weights[name] = t
    return weights


class PagedQwen3:
    """The decoder over packed tokens, its attention given by the caller. eight_bits:
    projections in 8 bits (embedding, norms, rotation and attention stay bf16)."""

    def __init__(self, shape: Qwen3Shape, weights: dict[str, torch.Tensor], max_positions: int, eight_bits: bool = False):
        self.shape, self.embed = shape, weights["model.embed_tokens.weight"]
        self.norm = weights["model.norm.weight"]
        self.lm_head = self.embed if shape.tied else weights["lm_head.weight"]
        self.layers = []
        for i in range(shape.layers):
            w = {k: weights[f"model.layers.{i}.{k}.weight"] for k in (
                "input_layernorm", "post_attention_layernorm", "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj",
                "self_attn.o_proj", "self_attn.q_norm", "self_attn.k_norm", "mlp.gate_proj", "mlp.up_proj", "mlp.down_proj")}
            w["qkv"] = torch.cat([w.pop(f"self_attn.{x}_proj") for x in "qkv"])
            w["gate_up"] = torch.cat([w.pop("mlp.gate_proj"), w.pop("mlp.up_proj")])
            if eight_bits:
                w |= {k: Fp8Weight(w[k]) for k in ("qkv", "self_attn.o_proj", "gate_up", "mlp.down_proj")}
            self.layers.append(w)
        self.eight_bits = eight_bits
        if eight_bits:
            self.lm_head = Fp8Weight(self.lm_head)
        inverse = 1.0 / shape.rope_theta ** (torch.arange(0, HEAD_DIM, 2, device="cuda").float() / HEAD_DIM)
        angle = torch.arange(max_positions, device="cuda").float()[:, None] * inverse
        self.cos, self.sin = (torch.cat([f(angle)] * 2, 1).bfloat16() for f in (torch.cos, torch.sin))

    def _rms(self, x, w):
        return w * (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + self.shape.eps)).bfloat16()

    def _rope(self, x, positions):
        half = HEAD_DIM // 2
        turned = torch.cat([-x[..., half:], x[..., :half]], -1)
        return x * self.cos[positions][:, None] + turned * self.sin[positions][:, None]

    def forward(self, tokens, positions, attend):
        """Logits of packed tokens; attend(layer, q, k, v) -> [tokens, q_heads, head_dim]."""
        if self.eight_bits:
            return self._forward_eight_bits(tokens, positions, attend)
        s = self.shape
        x = self.embed[tokens]
        for i, w in enumerate(self.layers):
            qkv = kernels.gemm_bt(self._rms(x, w["input_layernorm"]), w["qkv"])
            out = self._heads(i, w, qkv, positions, attend)
            x = x + kernels.gemm_bt(out, w["self_attn.o_proj"])
            gate, up = kernels.gemm_bt(self._rms(x, w["post_attention_layernorm"]), w["gate_up"]).chunk(2, 1)
            h = (torch.nn.functional.silu(gate.float()).bfloat16() * up).contiguous()
            x = x + kernels.gemm_bt(h, w["mlp.down_proj"])
        return kernels.gemm_bt(self._rms(x, self.norm), self.lm_head)

    def _heads(self, layer, w, qkv, positions, attend):
        """Norms and rotation of the heads, and their attention: [tokens, q_heads * head_dim]."""
        s = self.shape
        q, k, v = qkv.view(-1, s.q_heads + 2 * s.kv_heads, HEAD_DIM).split([s.q_heads, s.kv_heads, s.kv_heads], 1)
        q = self._rope(self._rms(q, w["self_attn.q_norm"]), positions)
        k = self._rope(self._rms(k, w["self_attn.k_norm"]), positions)
        return attend(layer, q, k, v.contiguous()).reshape(len(qkv), -1)

    def _forward_eight_bits(self, tokens, positions, attend):
        eps, x, residual = self.shape.eps, self.embed[tokens], None
        for i, w in enumerate(self.layers):
            residual, *rows = kernels.fp8_rms_norm(x, w["input_layernorm"], residual, eps, total=residual)
            out = self._heads(i, w, w["qkv"](rows), positions, attend)
            x = w["self_attn.o_proj"](kernels.fp8_quantize(out))
            residual, *rows = kernels.fp8_rms_norm(x, w["post_attention_layernorm"], residual, eps, total=residual)
            x = w["mlp.down_proj"](kernels.fp8_silu_multiply(w["gate_up"](rows)))
        return self.lm_head(kernels.fp8_rms_norm(x, self.norm, residual, eps, total=residual)[1:])


@dataclass
class Sampling:
    """How tokens are drawn (kernels.sample), for every sequence of a server."""

    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0


@dataclass
class Tree:
    """Drafted tokens of one step: node 0 is the newest token, a node's set its ancestors and itself."""

    tokens: list[int]
    parents: list[int] = field(default_factory=lambda: [-1])

    def child(self, node: int, token: int) -> int | None:
        return next((i for i in range(len(self.tokens)) if self.parents[i] == node and self.tokens[i] == token), None)

    def add(self, node: int, token: int) -> int:
        known = self.child(node, token)
        if known is not None:
            return known
        self.tokens.append(token)
        self.parents.append(node)
        return len(self.tokens) - 1

    def depths(self) -> list[int]:
        d: list[int] = []
        for p in self.parents:
            d.append(0 if p < 0 else d[p] + 1)
        return d

    def sets(self) -> list[int]:
        s: list[int] = []
        for i, p in enumerate(self.parents):
            s.append((s[p] if p >= 0 else 0) | 1 << i)
        return [x - (1 << 64) if x >> 63 else x for x in s]


def draft(text: list[int], width: int, depth: int) -> Tree:
    """Up to `width` continuations of `depth` tokens: what followed the newest token's last occurrences."""
    tree = Tree([text[-1]])
    found = 0
    for at in range(len(text) - 2, -1, -1):
        if found == width:
            break
        if text[at] != text[-1]:
            continue
        found += 1
        node = 0
        for token in text[at + 1:at + 1 + depth]:
            if len(tree.tokens) == 64:
                break
            node = tree.add(node, token)
    return tree


def _ints(values) -> torch.Tensor:
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def _starts(counts) -> list[int]:
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    return starts


class Server:
    def __init__(self, model: PagedQwen3, pages: int, page_size: int, sequences: int, max_positions: int,
                 sampling: Sampling | None = None):
        s = model.shape
        self.model, self.steps, self.emitted, self.sampling = model, 0, 0, sampling
        if sampling is not None:  # one random number for what follows each position of each sequence
            self.random = torch.Generator(device="cuda").manual_seed(sampling.seed)
            self.u = torch.rand(sequences, max_positions, device="cuda", generator=self.random)
            self.begun: set[int] = set()  # places whose numbers a sequence has had
        self.cache = KvCache(s.layers, pages, page_size, s.kv_heads, HEAD_DIM, sequences, max_positions)

    def _begin(self, sequences: list[int]) -> None:
        """Sequences begin in these places: where there was one before, with random numbers of their own."""
        if self.sampling is None:
            return
        again = [i for i in sequences if i in self.begun]
        if again:
            self.u[torch.tensor(again, device="cuda")] = torch.rand(len(again), self.u.shape[1], device="cuda", generator=self.random)
        self.begun.update(sequences)

    def choose(self, logits: torch.Tensor, sequences: list[int], positions: list[int]) -> list[int]:
        """The token after each row's position: the likeliest, or one drawn."""
        if self.sampling is None:
            return logits.argmax(-1).tolist()
        a, rows = self.sampling, len(sequences)
        last = self.u.shape[1] - 1  # a tree may be drafted past the room there is; the cache refuses such tokens
        u = self.u[torch.tensor(sequences, device="cuda"), torch.tensor([min(p, last) for p in positions], device="cuda")]
        full = lambda v, dtype=torch.float32: torch.full((rows,), v, dtype=dtype, device="cuda")  # noqa: E731
        tokens, _ = kernels.sample(logits, u, full(a.temperature), full(a.top_k, torch.int32), full(a.top_p), full(a.min_p))
        chosen = tokens.tolist()
        if min(chosen) < 0:
            raise RuntimeError("a row of logits has nothing to choose from, or the sampling's settings are out of range")
        return chosen

    def prefill(self, prompts: list[list[int]], sequences: list[int]) -> torch.Tensor:
        """Packed prompts into empty sequences; the logits after each."""
        s, cache = self.model.shape, self.cache
        self._begin(sequences)
        lens = [len(p) for p in prompts]
        plan = kernels.PromptPlan(lens, s.q_heads, s.kv_heads, HEAD_DIM)
        ids, starts = _ints(sequences), _starts(lens)
        offsets = _ints(starts)
        cache.extend(ids, offsets)

        def attend(layer, q, k, v):
            cache.write(layer, ids, offsets, k, v)
            return kernels.prompt_attention(plan, q, k, v)[0]

        tokens = torch.tensor([t for p in prompts for t in p], device="cuda")
        positions = torch.cat([torch.arange(n, device="cuda") for n in lens])
        return self.model.forward(tokens, positions, attend)[torch.tensor(starts[1:], device="cuda") - 1]

    def verify(self, texts: list[list[int]], sequences: list[int], trees: list[Tree], workspace) -> list[list[int]]:
        """One forward pass of every sequence's tree; appends what plain decoding would have
        taken to cache and texts, and returns the new tokens."""
        s, cache = self.model.shape, self.cache
        counts = [len(t.tokens) for t in trees]
        starts, ids = _starts(counts), _ints(sequences)
        offsets, sets = _ints(starts), torch.tensor([x for t in trees for x in t.sets()], device="cuda")
        held = torch.empty(2, s.layers, starts[-1], s.kv_heads, HEAD_DIM, dtype=torch.bfloat16, device="cuda")

        def attend(layer, q, k, v):
            held[0, layer], held[1, layer] = k, v
            return kernels.tree_attention(cache, layer, ids, offsets, sets, q, k, v, workspace)[0]

        tokens = torch.tensor([x for t in trees for x in t.tokens], device="cuda")
        places = [len(text) - 1 + d for text, t in zip(texts, trees) for d in t.depths()]
        logits = self.model.forward(tokens, torch.tensor(places, device="cuda"), attend)
        chosen = self.choose(logits, [i for i, n in zip(sequences, counts) for _ in range(n)], places)
        rows, taken, new = [], [], []
        for begin, text, tree in zip(starts, texts, trees):
            node, out, path = 0, [], []
            while node is not None:  # node's token stands; what follows it is known now
                path.append(begin + node)
                out.append(chosen[begin + node])
                node = tree.child(node, out[-1])
            rows += path
            taken.append(len(path))
            text += out
            new.append(out)
        cache.append(ids, _ints(_starts(taken)), held[0], held[1], _ints(rows))
        self.steps += 1
        self.emitted += sum(taken)
        return new

    def generate(self, prompts: list[list[int]], new_tokens: int, samples: int = 1, width: int = 4,
                 depth: int = 6) -> list[list[list[int]]]:
        """`samples` continuations of each prompt, of new_tokens tokens: drawn ones with a Sampling; else
        sample i begins with the prompt's i-th most likely next token and goes on greedily."""
        if not all(prompts):
            raise ValueError("a prompt needs at least one token")
        s, cache, many = self.model.shape, self.cache, len(prompts)
        logits = self.prefill(prompts, list(range(many)))
        owners = [p for p in range(many) for _ in range(samples)]
        if samples > 1:
            children = [many + i for i in range(many * (samples - 1))]
            cache.fork(_ints(p for p in range(many) for _ in range(samples - 1)), _ints(children))
            self._begin(children)
        slots = [p if i == 0 else many + p * (samples - 1) + i - 1 for p in range(many) for i in range(samples)]
        if self.sampling is None:
            first = logits.topk(samples, -1).indices.flatten().tolist()
        else:
            first = self.choose(logits.repeat_interleave(samples, 0), slots, [len(prompts[p]) - 1 for p in owners])
        texts = [list(prompts[p]) + [first[i]] for i, p in enumerate(owners)]
        live = list(range(len(texts)))
        workspace = kernels.tree_attention_workspace(len(texts), 64 * len(texts), s.q_heads, s.kv_heads, HEAD_DIM)
        while live:
            trees = [draft(texts[i], width, depth) for i in live]
            self.verify([texts[i] for i in live], [slots[i] for i in live], trees, workspace)
            done = [i for i in live if len(texts[i]) - len(prompts[owners[i]]) >= new_tokens]
            if done:
                cache.trim(_ints(slots[i] for i in done), _ints([0] * len(done)))
                cache.compact()
                live = [i for i in live if i not in done]
        if cache.status():
            raise RuntimeError("the cache refused a request: too few pages or positions")
        out: list[list[list[int]]] = [[] for _ in prompts]
        for i, p in enumerate(owners):
            out[p].append(texts[i][len(prompts[p]):][:new_tokens])
        return out


def main(argv=None) -> int:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--preset", choices=sorted(PRESETS), default="tiny")
    ap.add_argument("--seed", type=int, default=1234)
    ap.add_argument("--prompts", type=int, default=3)
    ap.add_argument("--prompt-len", type=int, default=64)
    ap.add_argument("--new-tokens", type=int, default=48)
    ap.add_argument("--samples", type=int, default=2)
    ap.add_argument("--width", type=int, default=4, help="drafted continuations a step, 0: plain decoding")
    ap.add_argument("--depth", type=int, default=6, help="tokens of each")
    ap.add_argument("--page-size", type=int, default=16)
    ap.add_argument("--eight-bits", action="store_true", help="projections in 8 bits")
    ap.add_argument("--temperature", type=float, help="draw tokens (default: the likeliest)")
    ap.add_argument("--top-k", type=int, default=0)
    ap.add_argument("--top-p", type=float, default=1.0)
    ap.add_argument("--min-p", type=float, default=0.0)
    a = ap.parse_args(argv)
    if a.temperature is None and (a.top_k, a.top_p, a.min_p) != (0, 1.0, 0.0):
        ap.error("--top-k, --top-p and --min-p need --temperature")
    shape = PRESETS[a.preset]
    room = a.prompt_len + a.new_tokens + a.depth + 2
    model = PagedQwen3(shape, synthetic_weights(shape, a.seed), room, a.eight_bits)
    sampling = None if a.temperature is None else Sampling(a.temperature, a.top_k, a.top_p, a.min_p, a.seed)
    sequences = a.prompts * a.samples
    server = Server(model, sequences * -(-room // a.page_size), a.page_size, sequences, room, sampling)
    g = torch.Generator().manual_seed(a.seed)
    prompts = [torch.randint(shape.vocab, (max(1, a.prompt_len - 7 * i),), generator=g).tolist() for i in range(a.prompts)]
    torch.cuda.synchronize()
    t = time.perf_counter()
    tokens = server.generate(prompts, a.new_tokens, a.samples, a.width, a.depth)
    torch.cuda.synchronize()
    print(json.dumps({"preset": a.preset, "sequences": sequences, "steps": server.steps, "seconds": round(time.perf_counter() - t, 3),
                      "tokens_per_step": round(server.emitted / max(1, server.steps) / sequences, 2), "generated_ids": tokens}))
    return 0


if __name__ == "__main__":
    raise SystemExit(main())
