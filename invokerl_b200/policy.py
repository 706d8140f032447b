"""PolicyModel with invokerl's interface (invokerl/policy.py:17-196) and the fused LM-head kernel.

`forward` keeps the reference's contract — per-token log-probs [B, T] with position 0 equal to
zero and position t holding log p(token_ids[t] | token_ids[<t]) — but the LM head + log-softmax +
gather run as one tcgen05 kernel that never materialises the [B*T, V] logits (the reference
loops over 64-token chunks under torch.utils.checkpoint).  Log-probs are returned in float32
(the reference returns the hidden dtype, bf16 by default).  Under FSDP the wrapped model still
produces full logits (policy.py:90-105); those go through the one-pass logits kernel instead of
F.cross_entropy.  Model loading, FSDP wrapping and vLLM weight sharing stay with the reference.
"""

from __future__ import annotations

import contextlib

import torch
from torch import Tensor

from . import ops


class PolicyModel:
    """Wraps a HuggingFace CausalLM; forward() returns per-token log-probs with gradients."""

    def __init__(
        self,
        model_name_or_path: str,
        device: str = "cuda",
        dtype: torch.dtype = torch.bfloat16,
        master_weights_fp32: bool = False,
    ):
        from transformers import AutoModelForCausalLM

        load_dtype = torch.float32 if master_weights_fp32 else dtype
        model = AutoModelForCausalLM.from_pretrained(model_name_or_path, dtype=load_dtype,
                                                     attn_implementation="sdpa").to(device)
        model.train()
        model.config.use_cache = False
        model.gradient_checkpointing_enable()
        self._setup(model, device, dtype, dtype if master_weights_fp32 else None)

    @classmethod
    def from_model(cls, model, device: str | torch.device = "cuda", dtype: torch.dtype = torch.bfloat16,
                   autocast_dtype: torch.dtype | None = None, fsdp_wrapped: bool = False) -> PolicyModel:
        """Wrap an already constructed CausalLM (no download)."""
        self = cls.__new__(cls)
        self._setup(model, device, dtype, autocast_dtype)
        self._fsdp_wrapped = fsdp_wrapped
        return self

    def _setup(self, model, device, dtype, autocast_dtype):
        self.model = model
        self.device = device
        self.dtype = dtype
        self.master_weights_fp32 = autocast_dtype is not None
        self._autocast_dtype = autocast_dtype
        self._fsdp_wrapped = False

    def forward(self, token_ids: Tensor, attention_mask: Tensor, ce_chunk_size: int = 64) -> Tensor:
        """Per-token log-probs [B, T] (fp32); position 0 is 0.  `ce_chunk_size` is accepted for
        interface compatibility; the fused kernel has no logits chunk to size."""
        token_ids = token_ids.to(self.device)
        attention_mask = attention_mask.to(self.device)
        ctx = (torch.autocast("cuda", dtype=self._autocast_dtype) if self._autocast_dtype
               else contextlib.nullcontext())
        with ctx:
            if self._fsdp_wrapped:
                logits = self.model(input_ids=token_ids, attention_mask=attention_mask).logits
                if logits.dtype != torch.bfloat16:
                    logits = logits.to(torch.bfloat16)
                # All T positions as rows of the [B*T, V] logits (a view, no copy of the slice
                # logits[:, :-1]); the last position has no target (-100, log-prob -0.0, no gradient).
                targets = torch.full_like(token_ids, -100)
                targets[:, :-1] = token_ids[:, 1:]
                log_probs = ops.logits_logprob(logits, targets)[:, :-1]
                pad = torch.zeros(token_ids.shape[0], 1, device=log_probs.device, dtype=log_probs.dtype)
                return torch.cat([pad, log_probs], dim=1)
            hidden = self.model.model(input_ids=token_ids, attention_mask=attention_mask).last_hidden_state
        # Every position t < T-1 predicts token t+1; the last position has no target (-100).
        targets = torch.full_like(token_ids, -100)
        targets[:, :-1] = token_ids[:, 1:]
        # Rows whose target is an attended token are the ones a loss can weight (the response
        # tokens among them); they are the candidates for the logit cache of the backward.
        cache_rows = torch.zeros_like(token_ids, dtype=torch.bool)
        cache_rows[:, :-1] = attention_mask[:, 1:].bool()
        lp = ops.lmhead_logprob(hidden, self.model.lm_head.weight, targets, cache_rows=cache_rows)
        pad = torch.zeros(token_ids.shape[0], 1, device=lp.device, dtype=lp.dtype)
        return torch.cat([pad, lp[:, :-1]], dim=1)

    def _chunked_lm_head_ce(self, hidden_states: Tensor, targets: Tensor, chunk_size: int) -> Tensor:
        """LM head + log-prob of `targets` for hidden_states [B, T, H] (policy.py:124-171); fp32."""
        return ops.lmhead_logprob(hidden_states, self.model.lm_head.weight, targets)

    @staticmethod
    def _chunk_ce_fn(lm_head_weight: Tensor, hidden_chunk: Tensor, target_chunk: Tensor) -> Tensor:
        """F.linear + -cross_entropy of one chunk (policy.py:173-191); fp32."""
        return ops.lmhead_logprob(hidden_chunk, lm_head_weight, target_chunk)

    # -- losses over token distributions (additions; the reference has none) ----------------------

    def _body(self, token_ids: Tensor, attention_mask: Tensor):
        """(logits, None) under FSDP, (None, last hidden states) otherwise."""
        ctx = (torch.autocast("cuda", dtype=self._autocast_dtype) if self._autocast_dtype
               else contextlib.nullcontext())
        with ctx:
            if self._fsdp_wrapped:
                return self.model(input_ids=token_ids, attention_mask=attention_mask).logits, None
            return None, self.model.model(input_ids=token_ids, attention_mask=attention_mask).last_hidden_state

    @staticmethod
    def _row_logits(logits: Tensor) -> Tensor:
        """Logits as the row losses and the top-k read them: bf16 and fp32 as they are, others in fp32."""
        return logits if logits.dtype in (torch.bfloat16, torch.float32) else logits.float()

    @staticmethod
    def _at_next_token(rows: Tensor) -> Tensor:
        """[B, T] row values (row t is about token t + 1) moved to the token they are about; 0 at position 0."""
        return torch.cat([torch.zeros_like(rows[:, :1]), rows[:, :-1]], dim=1)

    @torch.no_grad()
    def topk_log_probs(self, token_ids: Tensor, attention_mask: Tensor, k: int,
                       temperature: float = 1.0) -> tuple[Tensor, Tensor]:
        """As a teacher: (log_probs fp32, ids int64), both [B, T, k], where position t holds the k
        likeliest tokens given the tokens before t.  Position 0 and unattended positions hold no
        entries (-inf, -1), which `distill_loss` skips.  Without FSDP the logits are formed in bf16, as
        the model's own head gives them: log-probs carry that rounding (2^-8 of a logit), which the
        student's, summed in fp32 by the fused head, do not."""
        token_ids = token_ids.to(self.device)
        attention_mask = attention_mask.to(self.device)
        logits, hidden = self._body(token_ids, attention_mask)
        B, T = token_ids.shape
        log_probs = torch.full((B, T, k), -torch.inf, dtype=torch.float32, device=token_ids.device)
        ids = torch.full((B, T, k), -1, dtype=torch.int64, device=token_ids.device)
        if hidden is None:
            lp, top = ops.logits_topk(self._row_logits(logits), k, temperature)
            log_probs[:, 1:], ids[:, 1:] = lp[:, :-1], top[:, :-1]
        else:
            # logits of at most 1 GiB of rows at a time
            w = self.model.lm_head.weight.to(torch.bfloat16)
            h = hidden.to(torch.bfloat16)
            step = max(1, (1 << 30) // (2 * w.shape[0] * max(1, B)))
            for s in range(0, T - 1, step):
                e = min(s + step, T - 1)
                lp, top = ops.logits_topk(torch.nn.functional.linear(h[:, s:e], w), k, temperature)
                log_probs[:, s + 1:e + 1], ids[:, s + 1:e + 1] = lp, top
        off = ~attention_mask.bool()
        off[:, :1] = True
        return log_probs.masked_fill_(off[..., None], -torch.inf), ids.masked_fill_(off[..., None], -1)

    def distill_loss(self, token_ids: Tensor, attention_mask: Tensor, teacher_ids: Tensor, teacher_log_probs: Tensor,
                     kind: str = "forward", beta: float = 0.5, temperature: float = 1.0, tail: bool = True) -> Tensor:
        """Distillation loss of each token [B, T] (fp32; `ops.lmhead_distill`) against a teacher's
        entries [B, T, K] as `topk_log_probs` lays them out; position 0 is 0.  Weight it by the
        response mask: tokens whose loss has no gradient cost no backward work."""
        token_ids = token_ids.to(self.device)
        attention_mask = attention_mask.to(self.device)
        teacher_ids, teacher_log_probs = teacher_ids.to(self.device), teacher_log_probs.to(self.device)
        logits, hidden = self._body(token_ids, attention_mask)
        ids = torch.full_like(teacher_ids, -1)
        ids[:, :-1] = teacher_ids[:, 1:]
        lp = torch.roll(teacher_log_probs, -1, dims=1)
        args = (ids, lp, kind, beta, temperature, tail)
        if hidden is None:
            rows = ops.logits_distill(self._row_logits(logits), *args)
        else:
            rows = ops.lmhead_distill(hidden, self.model.lm_head.weight, *args)
        return self._at_next_token(rows)

    def cross_entropy_loss(self, token_ids: Tensor, attention_mask: Tensor, label_smoothing: float = 0.0,
                           z_loss: float = 0.0, loss_mask: Tensor | None = None) -> Tensor:
        """Cross entropy of each token [B, T] given the tokens before it (fp32;
        `ops.lmhead_cross_entropy`); 0 at position 0 and outside `loss_mask` (the attention mask by
        default)."""
        token_ids = token_ids.to(self.device)
        attention_mask = attention_mask.to(self.device)
        keep = attention_mask.bool() if loss_mask is None else loss_mask.to(self.device).bool()
        logits, hidden = self._body(token_ids, attention_mask)
        targets = torch.full_like(token_ids, -100)
        targets[:, :-1] = torch.where(keep[:, 1:], token_ids[:, 1:], -100)
        if hidden is None:
            rows = ops.logits_cross_entropy(self._row_logits(logits), targets, label_smoothing, z_loss)
        else:
            rows = ops.lmhead_cross_entropy(hidden, self.model.lm_head.weight, targets, label_smoothing, z_loss)
        return self._at_next_token(rows)

    @torch.no_grad()
    def forward_no_grad(self, token_ids: Tensor, attention_mask: Tensor) -> Tensor:
        """forward() without gradients (reference log-probs, policy.py:193-196)."""
        return self.forward(token_ids, attention_mask)
