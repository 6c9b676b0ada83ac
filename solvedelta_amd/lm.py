"""A minimal SolveDelta causal LM stack around the HIP mixer.

Just enough of the reference's model shell (causallsso/modeling_solvedelta.py:
31-100 MLP, :198-255 block, :283-395 model, :398-505 LM head and loss) to run
the CausalLM configuration end to end on MI355X and to capture its training
step in a HIP graph: token embedding, per layer pre-norm mixer + pre-norm
SwiGLU MLP with residuals, final norm, LM head and the shifted cross-entropy.
Module and parameter names follow the reference (``model.embeddings``,
``model.layers.{i}.mixer_norm / mixer.mixer / mlp_norm / mlp.gate_up_proj /
mlp.down_proj``, ``model.norm``, ``lm_head``) so its state dicts line up.
Norms, loss and, by default, the MLP are plain PyTorch-ROCm (hipBLASLt GEMMs);
``fused_ffn`` runs the MLP as one HIP operator (``gated_ffn``).  ``generate``
prefills, decodes token by token on the recurrent cache and draws each token
with ``sample_tokens``; ``quantize_linears`` puts a model's wide projections in 8
bits for it.  There is no hybrid attention here.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
import torch.nn.functional as F
from torch import nn

from .cache import RecurrentCache, SolveDeltaCacheAdapter
from .ffn import gated_ffn
from .mixer import SolveDeltaMixerConfig
from .sampling import Setting, sample_tokens


@dataclass
class SolveDeltaLMConfig(SolveDeltaMixerConfig):
    """Mixer fields plus the shell's (config.py:10-90)."""
    num_hidden_layers: int = 24
    hidden_ratio: Optional[int] = 4
    intermediate_size: Optional[int] = None
    vocab_size: int = 32000
    initializer_range: float = 0.02
    fused_ffn: bool = False


def _only_its_weight(proj: nn.Module) -> bool:
    """Whether calling ``proj`` is the product with its weight and nothing else."""
    return (type(proj) is nn.Linear and proj.bias is None and "forward" not in vars(proj)
            and not (proj._forward_hooks or proj._forward_pre_hooks or proj._backward_hooks
                     or proj._backward_pre_hooks))


class SolveDeltaMLP(nn.Module):
    """SwiGLU MLP with one gate/up projection (modeling_solvedelta.py:31-100).

    ``fused``: the whole block runs as ``gated_ffn``, in bf16 (parameters in bf16, or
    under bf16 autocast); projections that were put in 8 bits, have a bias, hooks or a
    forward of their own run on their own."""

    def __init__(self, hidden_size: int, hidden_ratio: Optional[int] = None,
                 intermediate_size: Optional[int] = None, fused: bool = False) -> None:
        super().__init__()
        if hidden_ratio is None:
            hidden_ratio = 4
        if intermediate_size is None:
            intermediate_size = int(hidden_size * hidden_ratio * 2 / 3)
            intermediate_size = 256 * ((intermediate_size + 255) // 256)
        self.hidden_size = hidden_size
        self.intermediate_size = intermediate_size
        self.fused = fused
        self.gate_up_proj = nn.Linear(hidden_size, 2 * intermediate_size, bias=False)
        self.down_proj = nn.Linear(intermediate_size, hidden_size, bias=False)

    def forward(self, x):
        if (self.fused and _only_its_weight(self.gate_up_proj) and _only_its_weight(self.down_proj)
                and not nn.modules.module._has_any_global_hook()):
            args = x, self.gate_up_proj.weight, self.down_proj.weight
            if x.is_cuda and torch.is_autocast_enabled("cuda"):
                dtype = torch.get_autocast_dtype("cuda")
                args = tuple(t.to(dtype) for t in args)
            return gated_ffn(*args)
        gate, value = self.gate_up_proj(x).chunk(2, dim=-1)
        return self.down_proj(F.silu(gate) * value)


class SolveDeltaBlock(nn.Module):
    def __init__(self, config: SolveDeltaLMConfig, layer_idx: int) -> None:
        super().__init__()
        self.layer_idx = layer_idx
        self.mixer_norm = nn.RMSNorm(config.hidden_size, eps=config.norm_eps)
        self.mixer = SolveDeltaCacheAdapter(config, layer_idx)
        self.mlp_norm = nn.RMSNorm(config.hidden_size, eps=config.norm_eps)
        self.mlp = SolveDeltaMLP(config.hidden_size, config.hidden_ratio,
                                 config.intermediate_size,
                                 fused=getattr(config, "fused_ffn", False))

    def forward(self, x, attention_mask=None, past_key_values=None, use_cache=False, **kw):
        y, _, past_key_values = self.mixer(self.mixer_norm(x), attention_mask=attention_mask,
                                           past_key_values=past_key_values, use_cache=use_cache,
                                           **kw)
        x = x + y
        return x + self.mlp(self.mlp_norm(x)), past_key_values


class SolveDeltaModel(nn.Module):
    def __init__(self, config: SolveDeltaLMConfig) -> None:
        super().__init__()
        self.config = config
        self.embeddings = nn.Embedding(config.vocab_size, config.hidden_size)
        self.layers = nn.ModuleList(SolveDeltaBlock(config, i)
                                    for i in range(config.num_hidden_layers))
        self.norm = nn.RMSNorm(config.hidden_size, eps=config.norm_eps)

    def forward(self, input_ids, attention_mask=None, past_key_values=None, use_cache=False,
                **kw):
        x = self.embeddings(input_ids)
        if use_cache and not isinstance(past_key_values, RecurrentCache):
            past_key_values = RecurrentCache.from_legacy_cache(past_key_values)
        elif not use_cache:
            past_key_values = None
        for layer in self.layers:
            x, past_key_values = layer(x, attention_mask=attention_mask,
                                       past_key_values=past_key_values, use_cache=use_cache, **kw)
        return self.norm(x), past_key_values


class SolveDeltaForCausalLM(nn.Module):
    def __init__(self, config: SolveDeltaLMConfig) -> None:
        super().__init__()
        self.config = config
        self.model = SolveDeltaModel(config)
        self.lm_head = nn.Linear(config.hidden_size, config.vocab_size, bias=False)
        self.apply(self._init_weights)

    def _init_weights(self, module):
        """Linear and embedding weights ~ N(0, initializer_range), biases zero
        (modeling_solvedelta.py:268-280); the mixer's own gate parameters keep
        their initial values."""
        if isinstance(module, nn.Linear):
            nn.init.normal_(module.weight, mean=0.0, std=self.config.initializer_range)
            if module.bias is not None:
                nn.init.zeros_(module.bias)
        elif isinstance(module, nn.Embedding):
            nn.init.normal_(module.weight, mean=0.0, std=self.config.initializer_range)

    def forward(self, input_ids, labels=None, attention_mask=None, past_key_values=None,
                use_cache: bool = False, **kw):
        """Returns (loss or None, logits, cache or None); the loss is the mean
        cross-entropy of token t+1 given tokens <= t (the last position ignored)."""
        h, cache = self.model(input_ids, attention_mask=attention_mask,
                              past_key_values=past_key_values, use_cache=use_cache, **kw)
        logits = self.lm_head(h)
        loss = None
        if labels is not None:
            shifted = torch.cat((labels[..., 1:], torch.full_like(labels[:, :1], -100)), dim=1)
            loss = F.cross_entropy(logits.reshape(-1, logits.shape[-1]).float(),
                                   shifted.reshape(-1), ignore_index=-100)
        return loss, logits, cache

    @torch.no_grad()
    def generate(self, input_ids, max_new_tokens: int, *, attention_mask=None,
                 temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                 min_p: Setting = 0.0, eos_token_id: Optional[int] = None,
                 pad_token_id: Optional[int] = None,
                 generator: Optional[torch.Generator] = None) -> torch.Tensor:
        """input_ids [B, T] and up to ``max_new_tokens`` more, int64 [B, T + new].

        One chunked pass over the prompt, then one decode step a token; each token
        is drawn from the last position's logits (``sample_tokens``; settings are
        numbers, or tensors with one entry per sequence; temperature 0 is greedy)
        with noise from ``generator``.  ``attention_mask`` [B, T] marks left padding.
        A sequence that drew ``eos_token_id`` goes on with ``pad_token_id`` (by default
        the end token itself, else 0), and the loop ends once all have; it looks
        every 16 tokens, since that waits for the GPU.  A sequence whose logits are
        all NaN ends the same way."""
        if input_ids.dim() != 2 or not input_ids.numel():
            raise ValueError("generate takes input_ids [B,T] with at least one token")
        if not isinstance(max_new_tokens, int) or max_new_tokens < 0:
            raise ValueError("max_new_tokens must be an int >= 0")
        if attention_mask is not None:
            if attention_mask.shape != input_ids.shape:
                raise ValueError("attention_mask must have the shape of input_ids")
            if not bool(attention_mask[:, -1].all()):
                raise ValueError("generate takes left-padded prompts")
        batch, length = input_ids.shape
        pad = pad_token_id if pad_token_id is not None else (eos_token_id or 0)
        out = input_ids.new_full((batch, length + max_new_tokens), pad)
        out[:, :length] = input_ids
        done = torch.zeros(batch, dtype=torch.bool, device=input_ids.device)
        cache, ids, mask = RecurrentCache(), input_ids, attention_mask
        for i in range(max_new_tokens):
            h, cache = self.model(ids, attention_mask=mask, past_key_values=cache, use_cache=True)
            logits, mask = self.lm_head(h[:, -1]), None
            noise = torch.rand(logits.shape, dtype=torch.float32, device=logits.device,
                               generator=generator)
            token = sample_tokens(logits, noise, temperature, top_k, top_p, min_p)
            done |= token < 0
            token.masked_fill_(done, pad)
            out[:, length + i] = token
            if eos_token_id is not None:
                done |= token == eos_token_id
            if i % 16 == 15 and bool(done.all()):
                return out[:, :length + i + 1]
            ids = token.unsqueeze(1)
        return out


__all__ = ["SolveDeltaLMConfig", "SolveDeltaMLP", "SolveDeltaBlock", "SolveDeltaModel",
           "SolveDeltaForCausalLM"]
