"""Greedy decoding of a batch of requests over one paged cache: the batch operators together.

``UnifiedEngine`` decodes one sequence; ``BatchDecoder`` runs the same decoder (preq2 W4A8
projections, partial rotary embedding, int8 cache, grouped heads) for several requests at once:

    dec = BatchDecoder(model, max_requests=8, pages=512, page_size=16, window=1024, sinks=4)
    out = dec.generate(prompts, 32, repetition=1.1, mask=grammar_bits)

Every step builds its plan on the GPU (``plan_step``), writes the new keys and values through the slot
map (``kv_write``), attends over the pages (``attention_paged`` with the window and sinks, or
``attention_shared_prefix`` when the requests share a prefix) and applies penalties, biases and the
grammar mask to the logits (``logits_process``).  Prompts go in as one ragged step, then one token per
request and step.  The projections are the multi-token GEMVs (``asdsl_b200_gemv_multi``); norms,
rotation and SiLU are plain torch: this shows the operators in use, the decode engine is the tuned
path for one sequence.
"""

from __future__ import annotations

import numpy as np
import torch

from asdsl_b200 import _lib
from asdsl_b200.kernels import (
    AttentionWorkspace,
    PagedKV,
    StepPlan,
    attention_paged,
    attention_shared_prefix,
    kv_write,
    logits_process,
    plan_step,
)
from asdsl_b200.quantization.device import prepare_preq2_device


def _cuda(a) -> torch.Tensor:
    return a.cuda() if isinstance(a, torch.Tensor) else torch.from_numpy(np.ascontiguousarray(a)).cuda()


class BatchDecoder:
    """Decoder of a synthetic model (asdsl_b200.inference.synthetic.build_model) for up to max_requests
    requests with `pages` pages of page_size positions per layer.  window = 0: every position is seen.
    lm_head: preq2 (meta, quant), as the decode engine exports it (export_lm_head_preq2); by default
    the tied embedding is quantized here."""

    def __init__(self, model: dict, max_requests: int, pages: int, page_size: int = 16, window: int = 0, sinks: int = 0,
                 cache_dtype=torch.int8, attention_dtype=torch.float16, lm_head=None):
        c = self.config = model["config"]
        self.window, self.sinks, self.page_size, self.pages = window, sinks, page_size, pages
        self.attention_dtype = attention_dtype
        self.embed = _cuda(model["embed_f16"]).view(torch.float16)
        self.cos, self.sin = _cuda(model["cos"]), _cuda(model["sin"])
        self.out_norm = _cuda(model["output_norm"])
        self.layers = [{k: _cuda(v) for k, v in layer.items()} for layer in model["layers"]]
        self.caches = [PagedKV.empty(pages, page_size, c["n_kv_heads"], c["head_dim"], cache_dtype) for _ in self.layers]
        if lm_head is None:
            lm_head = prepare_preq2_device(self.embed.float())
        self.lm_head = {"lm_head_meta": _cuda(lm_head[0]), "lm_head_quant": _cuda(lm_head[1])}
        self.max_requests = max_requests
        self.free = torch.arange(pages, dtype=torch.int32, device="cuda")
        self.taken = 0  # pages handed out so far, from the front of `free`
        self.workspace = AttentionWorkspace()

    # ---- the layers ----

    def _gemv(self, layer: dict, name: str, x: torch.Tensor, rows: int) -> torch.Tensor:
        y = torch.empty(x.shape[0], rows, dtype=torch.float32, device="cuda")
        _lib.call("asdsl_b200_gemv_multi", _lib.FMT_PREQ2, layer[name + "_meta"].data_ptr(), layer[name + "_quant"].data_ptr(),
                  x.contiguous().data_ptr(), y.data_ptr(), rows, x.shape[1], x.shape[0], torch.cuda.current_stream().cuda_stream)
        return y

    def _norm(self, x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + self.config["eps"]) * w

    def _rotate(self, x: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        half = self.config["rotary_dim"] // 2
        cos, sin = self.cos[positions][:, None], self.sin[positions][:, None]
        a, b = x[..., :half], x[..., half : 2 * half]
        return torch.cat([a * cos - b * sin, a * sin + b * cos, x[..., 2 * half :]], -1)

    def _forward(self, tokens: torch.Tensor, plan: StepPlan, ragged: bool, prefix) -> torch.Tensor:
        """Hidden states of the step's tokens [t, hidden]; their keys and values go to the pages."""
        c = self.config
        heads, kvh, d, t = c["n_heads"], c["n_kv_heads"], c["head_dim"], tokens.numel()
        before = 0 if prefix is None else prefix[1]
        positions = (plan.positions[:t] + before).long()
        cu = plan.cu_q if ragged else None
        x = self.embed[tokens.long()].float()
        for layer, cache in zip(self.layers, self.caches):
            qkv = self._gemv(layer, "qkv_proj", self._norm(x, layer["rms_att"]), (heads + 2 * kvh) * d).view(t, heads + 2 * kvh, d)
            q = self._rotate(qkv[:, :heads], positions).to(self.attention_dtype)
            kv_write(cache, self._rotate(qkv[:, heads : heads + kvh], positions), qkv[:, heads + kvh :].contiguous(), plan.slots)
            if prefix is None:
                o = attention_paged(q, cache, plan.block_table, plan.total_lens, cu, window=self.window, sinks=self.sinks,
                                    workspace=self.workspace)
            else:
                o = attention_shared_prefix(q, cache, prefix[0], prefix[1], plan.block_table, plan.total_lens, cu,
                                            workspace=self.workspace)
            x = x + self._gemv(layer, "o_proj", o.float().view(t, heads * d), c["hidden"])
            gu = self._gemv(layer, "gate_up_proj", self._norm(x, layer["rms_ffn"]), 2 * c["inter"])
            x = x + self._gemv(layer, "down_proj", torch.nn.functional.silu(gu[:, : c["inter"]]) * gu[:, c["inter"] :], c["hidden"])
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return self._gemv(self.lm_head, "lm_head", self._norm(x, self.out_norm), self.config["vocab"])

    # ---- a batch ----

    def _step(self, plan: StepPlan, held: list[int], new: list[int], tokens: torch.Tensor, prefix) -> torch.Tensor:
        pages = sum(-(-(a + b) // self.page_size) - -(-a // self.page_size) for a, b in zip(held, new))
        if self.taken + pages > self.pages:
            raise RuntimeError(f"the cache's {self.pages} pages are taken")
        lens = torch.tensor([held, new], dtype=torch.int32).cuda(non_blocking=True)
        plan_step(plan, lens[0], lens[1], self.free[self.taken :])
        self.taken += pages
        return self._forward(tokens, plan, max(new) > 1, prefix)

    def reset(self) -> None:
        """Every page is free again."""
        self.taken = 0

    def generate(self, prompts: list[list[int]], n_new: int, prefix: list[int] | None = None, repetition: float = 1.0,
                 frequency: float = 0.0, presence: float = 0.0, biases: dict[int, float] | None = None,
                 mask: torch.Tensor | None = None, logits_out: list | None = None) -> list[list[int]]:
        """n_new greedy tokens after each prompt.  prefix: tokens that come before every prompt, held once and
        part of each request's history for the penalties, not of what is returned (every row sees all of
        it, so a decoder with a window refuses one); mask: int32 [ceil(vocab / 32)] bits
        of the allowed ids; logits_out collects each step's processed logits."""
        n, vocab = len(prompts), self.config["vocab"]
        if not 0 < n <= self.max_requests or any(not p for p in prompts):
            raise ValueError(f"1 to {self.max_requests} prompts that are not empty")
        if prefix and self.window > 0:
            raise ValueError("a shared prefix is attended without a window: give the joined prompts, or a decoder of window 0")
        longest = max(map(len, prompts)) + n_new
        before = list(prefix or [])
        if longest + len(before) > self.config["max_seq"]:
            raise ValueError("prompt and new tokens exceed the model's positions")
        shared = None
        if prefix:
            pre = StepPlan(1, len(prefix), -(-len(prefix) // self.page_size), self.page_size)
            self._step(pre, [0], [len(prefix)], torch.tensor(prefix, dtype=torch.int32, device="cuda"), None)
            shared = (pre.block_table[0], len(prefix))
        plan = StepPlan(n, sum(map(len, prompts)), -(-longest // self.page_size), self.page_size)
        history = torch.zeros(n, len(before) + longest, dtype=torch.int32, device="cuda")
        for b, p in enumerate(prompts):
            history[b, : len(before) + len(p)] = torch.tensor(before + list(p), dtype=torch.int32)
        prompt_lens = torch.tensor([len(before) + len(p) for p in prompts], dtype=torch.int32, device="cuda")
        ones = torch.ones(n, device="cuda")
        bias = {}
        if biases:
            ids, values = list(biases), list(biases.values())
            bias = dict(bias_ptr=torch.arange(n + 1, dtype=torch.int32, device="cuda") * len(ids),
                        bias_ids=torch.tensor(ids * n, dtype=torch.int32, device="cuda"),
                        bias_values=torch.tensor(values * n, dtype=torch.float32, device="cuda"))
        bits = None if mask is None else mask.cuda()[None].expand(n, -1)
        held, new = [0] * n, [len(p) for p in prompts]
        tokens = torch.cat([torch.tensor(p, dtype=torch.int32) for p in prompts]).cuda()
        for step in range(n_new):
            x = self._step(plan, held, new, tokens, shared)
            last = plan.cu_q[1:].long() - 1
            held, new = [a + b for a, b in zip(held, new)], [1] * n
            lens = prompt_lens + step
            logits = logits_process(self._logits(x[last]), tokens=history, lens=lens, prompt_lens=prompt_lens,
                                    repetition=ones * repetition, frequency=ones * frequency, presence=ones * presence,
                                    mask=bits, **bias)
            if logits_out is not None:
                logits_out.append(logits)
            tokens = logits.argmax(-1).to(torch.int32)
            history.scatter_(1, lens.long()[:, None], tokens[:, None])
        return [history[b, len(before) : len(before) + len(p) + n_new].tolist() for b, p in enumerate(prompts)]
