"""A batch of prompts and its next tokens through one decoder layer: the operators for packed sequences
together, as a server would drive them.

The prompts go in as one packed call: embedding -> rmsnorm -> matmul x3 -> rope-axes x2 -> kv-write-packed x2
(the keys and values into 4-bit stores, a slot of rows for each sequence) -> attention-packed over the prompts' own
keys -> matmul-residual -> rmsnorm -> gated-matmul -> matmul-residual -> rmsnorm -> matmul (logits) ->
token-logprobs of the tokens that follow.  A step has one token of each sequence: the same nodes, with attention
over the stores; ``capture`` records them once, with the key counts advancing, and each step is one replay.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, List, Sequence, Tuple

import numpy as np

from .executor import CudaExecutor, KernelInvocation
from .layer import DecoderLayerConfig


@dataclass(frozen=True)
class PackedBatchConfig(DecoderLayerConfig):
    kv_heads: int = 4
    sections: Tuple[int, ...] = (12, 10, 10)  # rotary pairs of each position axis (time, height, width)
    slot: int = 1024                          # rows a sequence has in the stores
    top: int = 1                              # alternatives reported with each token


WEIGHTS = ("table", "attn_norm", "wq", "wk", "wv", "wo", "mlp_norm", "wg", "wu", "wd", "final_norm", "head")


def make_weights(cfg: PackedBatchConfig, seed: int = 0) -> Dict[str, np.ndarray]:
    """Seeded synthetic weights N(0, std); the norms' around one."""
    rng = np.random.default_rng(seed)
    h, f, q, kv = cfg.hidden, cfg.ffn, cfg.heads * cfg.head_dim, cfg.kv_heads * cfg.head_dim
    shapes = {"table": (cfg.vocab, h), "attn_norm": (h,), "wq": (h, q), "wk": (h, kv), "wv": (h, kv), "wo": (q, h),
              "mlp_norm": (h,), "wg": (h, f), "wu": (h, f), "wd": (f, h), "final_norm": (h,), "head": (h, cfg.vocab)}
    w = {n: (rng.standard_normal(s, dtype=np.float32) * cfg.weight_std).astype(np.float32) for n, s in shapes.items()}
    for n in ("attn_norm", "mlp_norm", "final_norm"):
        w[n] += 1
    return w


def invocations(cfg: PackedBatchConfig, prefix: str, write_table: str, keys: str, values: str, read_table: str,
                scored: bool) -> List[KernelInvocation]:
    """The nodes over the packed rows ``prefix`` + "ids" at ``prefix`` + "positions": keys and values written
    into "key_store" and "value_store" by ``write_table``, attention over ``keys`` and ``values`` by ``read_table``;
    ``scored``: log probabilities of ``prefix`` + "targets"."""
    p = prefix
    inv = KernelInvocation

    def rope(heads):
        return {"base": float(cfg.rope_theta), "dimension": cfg.head_dim, "head_count": heads, "rotation_pairing": "half_split",
                "sections": ",".join(str(s) for s in cfg.sections), "section_order": "cyclic"}

    eps = {"epsilon": float(cfg.eps)}
    return [
        inv("embedding", ["table", p + "ids"], p + "x"),
        inv("rmsnorm", [p + "x", "attn_norm"], p + "h", eps),
        inv("matmul", [p + "h", "wq"], p + "q"),
        inv("matmul", [p + "h", "wk"], p + "k"),
        inv("matmul", [p + "h", "wv"], p + "v"),
        inv("rope-axes", [p + "q", p + "positions"], p + "qr", rope(cfg.heads)),
        inv("rope-axes", [p + "k", p + "positions"], p + "kr", rope(cfg.kv_heads)),
        inv("kv-write-packed", ["key_store", p + "kr", write_table], "key_store"),
        inv("kv-write-packed", ["value_store", p + "v", write_table], "value_store"),
        inv("attention-packed", [p + "qr", keys, values, read_table], p + "a",
            {"head_count": cfg.heads, "head_dimension": cfg.head_dim, "kv_head_count": cfg.kv_heads, "causal": True}),
        inv("matmul-residual", [p + "a", "wo", p + "x"], p + "x2"),
        inv("rmsnorm", [p + "x2", "mlp_norm"], p + "h2", eps),
        inv("gated-matmul", [p + "h2", "wg", "wu"], p + "g"),
        inv("matmul-residual", [p + "g", "wd", p + "x2"], p + "out"),
        inv("rmsnorm", [p + "out", "final_norm"], p + "hf", eps),
        inv("matmul", [p + "hf", "head"], p + "logits"),
        inv("token-logprobs", [p + "logits"] + ([p + "targets"] if scored else []), p + "scores", {"top": cfg.top}),
    ]


class PackedBatch:
    """One batch on one executor: ``prefill``, ``capture``, then a ``step`` for each further token."""

    def __init__(self, ex: CudaExecutor, cfg: PackedBatchConfig, weights: Dict[str, np.ndarray]):
        if sum(cfg.sections) * 2 != cfg.head_dim:
            raise ValueError(f"sections {cfg.sections} do not make up the {cfg.head_dim // 2} pairs of a head")
        self.ex, self.cfg, self.lengths, self.steps, self._replay = ex, cfg, [], 0, None
        for name in WEIGHTS:
            ex.write_weight_tensor(name, weights[name])

    def _positions(self, positions, starts, counts) -> np.ndarray:
        """[rows, axes]; without positions of its own a token stands at its index on every axis (text)."""
        if positions is None:
            positions = np.concatenate([np.arange(s, s + n) for s, n in zip(starts, counts)])[:, None].repeat(len(self.cfg.sections), 1)
        return np.ascontiguousarray(positions, np.float32)

    def prefill(self, prompts: Sequence[np.ndarray], positions=None) -> np.ndarray:
        """Runs the prompts and keeps their keys and values; returns [tokens, 2 + 2 top]: of each token's
        successor in its prompt the log probability (NaN for the last), the entropy, the top alternatives."""
        ex, cfg, n = self.ex, self.cfg, [len(p) for p in prompts]
        if not n or min(n) == 0:
            raise ValueError(f"a batch needs prompts of at least one token each, got lengths {n}")
        if max(n) >= cfg.slot:
            raise ValueError(f"a prompt of {max(n)} tokens leaves no room in a slot of {cfg.slot}")
        self.lengths, self.steps, self._replay = list(n), 0, None
        ks = ex.kernels
        starts = [i * cfg.slot for i in range(len(n))]
        for name in ("key_store", "value_store"):
            ex.adopt(name, ks.kv_store_q4(cfg.slot * len(n), cfg.kv_heads, cfg.head_dim))
        ex.adopt("prompts", ks.sequences(n))
        ex.adopt("slots", ks.sequences(n, n, starts))
        ex.adopt("next", ks.sequences([1] * len(n), [m + 1 for m in n], starts))
        ex.write_tensor("p.ids", np.concatenate(prompts).astype(np.float32))
        ex.write_tensor("p.positions", self._positions(positions, [0] * len(n), n))
        ex.write_tensor("p.targets", np.concatenate([np.append(p[1:], -1) for p in prompts]).astype(np.float32))
        for node in invocations(cfg, "p.", "slots", "p.kr", "p.v", "prompts", scored=True):
            ex.run(node)
        return ex.read_tensor("p.scores")

    def capture(self) -> None:
        """Records a step.  (The rows that the recorded run writes are those that the first step writes again.)"""
        if not self.lengths or self.steps:
            raise RuntimeError("a step is captured after prefill and before the first step, whose rows the recorded run writes")
        ex, b = self.ex, len(self.lengths)
        self._ids, self._at = np.zeros(b, np.float32), np.zeros((b, len(self.cfg.sections)), np.float32)
        self._scores = np.empty((b, 2 + 2 * self.cfg.top), np.float32)
        ex.write_tensor("s.ids", self._ids)
        ex.write_tensor("s.positions", self._at)
        nodes = invocations(self.cfg, "s.", "next", "key_store", "value_store", "next", scored=False)
        for node in nodes:
            ex.run(node)
        ex.synchronize()
        ex.begin_step_capture(["key_count"])
        try:
            for node in nodes:
                ex.run(node)
        except Exception:
            ex.abort_step_capture()
            raise
        ex.end_step_capture()
        self._replay = ex.step_io({"s.ids": self._ids, "s.positions": self._at}, {"s.scores": self._scores})

    def step(self, ids: Sequence[int], positions=None) -> np.ndarray:
        """One more token of each sequence: [sequences, 2 + 2 top], the likeliest next tokens in the last
        ``top`` columns.  A step past the end of a slot is refused."""
        if self._replay is None:
            raise RuntimeError("a step needs capture() after the prefill")
        self._ids[:] = ids
        self._at[:] = self._positions(positions, [n + self.steps for n in self.lengths], [1] * len(self.lengths))
        self._replay(self.steps)
        self.steps += 1
        return self._scores

    def generate(self, scores: np.ndarray, steps: int) -> List[List[int]]:
        """The likeliest continuation, from the scores of the prefill (or of the last step)."""
        if self.cfg.top < 1:
            raise ValueError("the likeliest tokens are among the alternatives: top is 0")
        top = scores[np.cumsum(self.lengths) - 1] if len(scores) != len(self.lengths) else scores
        tokens: List[List[int]] = [[] for _ in self.lengths]
        for _ in range(steps):
            ids = top[:, 2 + self.cfg.top].astype(int)
            for t, i in zip(tokens, ids):
                t.append(int(i))
            top = self.step(ids)
        return tokens
