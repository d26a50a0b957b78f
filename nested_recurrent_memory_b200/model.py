"""Full-model forward harness: the NestedGDN-2 language model around this
package's op (the caller side of the hot path).

A plain-torch restatement of the reference's layer and model,
nested_gdn2/layers/nested_gdn2.py:28-237 (``NestedGDN2Attention``) and
nested_gdn2/models/modeling_nested_gdn2.py:43-160 (block, model, LM head),
with the same parameter names and shapes so that a reference state dict
loads unchanged. fla's modules that the reference imports are restated from
their published definitions: ``ShortConvolution`` (depthwise causal
convolution with SiLU), ``RMSNorm``, ``FusedRMSNormGated`` (RMSNorm times a
sigmoid gate) and ``GatedMLP`` (SwiGLU, intermediate size
256 * ceil(hidden * ratio * 2/3 / 256)). Dense layers run as torch (cuBLAS)
GEMMs; the token mixer's op is ``chunk_nested_gdn2`` from this package
(hand-written sm_100a kernels) unless another op with the same signature is
passed in. No decode cache for the nested layers.

Beyond the reference, the embedding may scale its rows (``embed_tokens``), and
the layers named in ``recurrent_layers`` mix tokens with the channel-wise
gated recurrence (``gated_scan``) instead of the nested op. A model of such
layers only decodes token by token (``NestedGDN2ForCausalLM.step``). The forward
is differentiable, so the same module trains (see ``optim.Muon``); ``step`` is
not.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch
import torch.nn as nn
import torch.nn.functional as F

from .embedding import embed_tokens
from .ops import _DTYPES, chunk_nested_gdn2
from .recurrence import gated_scan, step_gated_scan

__all__ = ["ModelConfig", "NestedGDN2Attention", "GatedRecurrence", "ScaledEmbedding",
           "NestedGDN2Block", "NestedGDN2ForCausalLM"]


# Whether a tensor is torch.func's stand-in for one, without memory of its own.
_is_transformed = torch._C._functorch.is_functorch_wrapped_tensor


@dataclass
class ModelConfig:
    """The fields of NestedGDN2Config (configuration_nested_gdn2.py:14-47)
    that the forward reads; defaults are BASELINE config 4's."""
    vocab_size: int = 32000
    hidden_size: int = 1024
    num_hidden_layers: int = 12
    num_heads: int = 8
    head_dim: int = 128
    expand_v: float = 1.0
    conv_size: int = 4
    hidden_ratio: int = 4
    intermediate_size: int | None = None
    norm_eps: float = 1e-5
    initializer_range: float = 0.02
    num_levels: int = 3
    firing_intervals: tuple = (1, 4, 16)
    n_queries_per_level: tuple = field(default_factory=lambda: (64, 64))
    promotion: str = "learned"
    read_mix: str = "softmax"
    max_horizon: int | None = None
    embed_scale: float = 1.0
    recurrent_layers: tuple = ()  # indices of the layers that mix by GatedRecurrence


class ShortConvolution(nn.Module):
    """Depthwise causal 1-D convolution over time followed by SiLU (fla's
    ShortConvolution with activation="silu", no bias)."""

    def __init__(self, channels: int, kernel_size: int):
        super().__init__()
        self.kernel_size = kernel_size
        self.weight = nn.Parameter(torch.empty(channels, 1, kernel_size))

    def forward(self, x):  # [B, T, C]
        T = x.shape[1]
        y = F.conv1d(x.transpose(1, 2), self.weight, padding=self.kernel_size - 1,
                     groups=self.weight.shape[0])[..., :T]
        return F.silu(y).transpose(1, 2)


class RMSNorm(nn.Module):
    def __init__(self, dim: int, eps: float):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(dim))

    def forward(self, x):
        xf = x.float()
        y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + self.eps)
        return (y * self.weight.float()).to(x.dtype)


class GatedRMSNorm(RMSNorm):
    """RMSNorm over the last dimension times sigmoid(gate) (fla's
    FusedRMSNormGated with activation="sigmoid")."""

    def forward(self, x, gate):
        return (super().forward(x).float() * torch.sigmoid(gate.float())).to(x.dtype)


class GatedMLP(nn.Module):
    """SwiGLU channel mixer (fla's GatedMLP, hidden_act="swish")."""

    def __init__(self, hidden: int, ratio: int, intermediate: int | None):
        super().__init__()
        if intermediate is None:
            intermediate = int(hidden * ratio * 2 / 3)
            intermediate = 256 * ((intermediate + 255) // 256)
        self.gate_proj = nn.Linear(hidden, intermediate, bias=False)
        self.up_proj = nn.Linear(hidden, intermediate, bias=False)
        self.down_proj = nn.Linear(intermediate, hidden, bias=False)

    def forward(self, x):
        return self.down_proj(F.silu(self.gate_proj(x)) * self.up_proj(x))


class NestedGDN2Attention(nn.Module):
    """The token-mixing layer (nested_gdn2.py:28-237), short convolutions on."""

    def __init__(self, cfg: ModelConfig, op=None):
        super().__init__()
        self.cfg = cfg
        self.op = op or chunk_nested_gdn2
        self.L = L = cfg.num_levels
        H, K = cfg.num_heads, cfg.head_dim
        V = int(cfg.head_dim * cfg.expand_v)
        self.H, self.K, self.V = H, K, V
        self.key_dim, self.value_dim = H * K, H * V
        d = cfg.hidden_size
        self.q_proj = nn.Linear(d, L * self.key_dim, bias=False)
        self.k_proj = nn.Linear(d, self.key_dim, bias=False)
        self.v_proj = nn.Linear(d, self.value_dim, bias=False)
        self.q_conv1d = ShortConvolution(L * self.key_dim, cfg.conv_size)
        self.k_conv1d = ShortConvolution(self.key_dim, cfg.conv_size)
        self.v_conv1d = ShortConvolution(self.value_dim, cfg.conv_size)
        self.f_proj = nn.Sequential(nn.Linear(d, V, bias=False), nn.Linear(V, self.key_dim, bias=False))
        self.b_proj = nn.Linear(d, self.key_dim, bias=False)
        self.w_proj = nn.Linear(d, self.value_dim, bias=False)
        # nested_gdn2.py:66-71
        self.A_log = nn.Parameter(torch.log(torch.empty(H, dtype=torch.float32).uniform_(1, 16)))
        dt = torch.exp(torch.rand(self.key_dim) * (math.log(0.1) - math.log(0.001))
                       + math.log(0.001)).clamp(min=1e-4)
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        # nested_gdn2.py:73-92
        n_max = max(cfg.n_queries_per_level) if L > 1 else 1
        self.b_projections = nn.Parameter(torch.randn(L - 1, H, V, K) * V ** -0.5)
        self.w_projections = nn.Parameter(torch.randn(L - 1, H, V, V) * V ** -0.5)
        self.g_projections = nn.Parameter(torch.randn(L - 1, H, V, K) * V ** -0.5)
        self.query_banks = nn.Parameter(torch.randn(L - 1, H, n_max, K) * K ** -0.5)
        self.key_projections = nn.Parameter(torch.randn(L - 1, H, K, V) * V ** -0.5)
        self.n_queries_per_level = tuple(cfg.n_queries_per_level)
        self.firing_intervals = tuple(cfg.firing_intervals)
        self.mix_proj = nn.Linear(d, H * L, bias=False)
        self.g_proj = nn.Sequential(nn.Linear(d, V, bias=False), nn.Linear(V, self.value_dim, bias=True))
        self.o_norm = GatedRMSNorm(V, cfg.norm_eps)
        self.o_proj = nn.Linear(self.value_dim, d, bias=False)

    def forward(self, x, initial_state=None):
        """x [B, T, d] -> (output [B, T, d], final state [B, H, L, K, V])."""
        B, T, _ = x.shape
        H, K, V, L = self.H, self.K, self.V, self.L
        q = self.q_conv1d(self.q_proj(x)).reshape(B, T, L, H, K).transpose(2, 3)
        k = self.k_conv1d(self.k_proj(x)).reshape(B, T, H, K)
        v = self.v_conv1d(self.v_proj(x)).reshape(B, T, H, V)
        q = F.normalize(q, dim=-1).to(v.dtype)
        k = F.normalize(k, dim=-1).to(v.dtype)
        # nested_gdn2.py:142-150: per-channel log-decay in fp32, gates.
        g0 = F.softplus(self.f_proj(x).float() + self.dt_bias).reshape(B, T, H, K)
        g0 = -self.A_log.float().exp()[:, None] * g0
        if self.cfg.max_horizon:
            g0 = g0.clamp(max=-1.0 / self.cfg.max_horizon)
        b0 = self.b_proj(x).sigmoid().reshape(B, T, H, K)
        w0 = self.w_proj(x).sigmoid().reshape(B, T, H, V)
        logits = self.mix_proj(x).reshape(B, T, H, L)
        mix = (logits.sigmoid() if self.cfg.read_mix == "sigmoid" else logits.softmax(-1)).to(v.dtype)
        o, state = self.op(
            q=q, k=k, v=v, g=g0, b=b0, w=w0, mix_weights=mix,
            query_banks=self.query_banks, key_projections=self.key_projections,
            b_projections=self.b_projections, w_projections=self.w_projections,
            g_projections=self.g_projections, n_queries_per_level=self.n_queries_per_level,
            firing_intervals=self.firing_intervals, L=L, initial_state=initial_state,
            output_final_state=True, chunk_size=64, promotion=self.cfg.promotion)
        o = self.o_norm(o, self.g_proj(x).reshape(B, T, H, V))
        return self.o_proj(o.reshape(B, T, H * V)), state


class GatedRecurrence(nn.Module):
    """A token mixer of one gated linear recurrence a channel,
    h_t = e^{g_t} h_{t-1} + sqrt(1 - e^{2 g_t}) v_t, with the nested layer's
    decay parameterisation and gated output norm. Its state is [B, value_dim]
    float32."""

    def __init__(self, cfg: ModelConfig):
        super().__init__()
        d, self.H, self.V = cfg.hidden_size, cfg.num_heads, int(cfg.head_dim * cfg.expand_v)
        width = self.H * self.V
        self.v_proj = nn.Linear(d, width, bias=False)
        self.f_proj = nn.Sequential(nn.Linear(d, self.V, bias=False), nn.Linear(self.V, width, bias=False))
        self.A_log = nn.Parameter(torch.log(torch.empty(width, dtype=torch.float32).uniform_(1, 16)))
        dt = torch.exp(torch.rand(width) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.g_proj = nn.Sequential(nn.Linear(d, self.V, bias=False), nn.Linear(self.V, width, bias=True))
        self.o_norm = GatedRMSNorm(self.V, cfg.norm_eps)
        self.o_proj = nn.Linear(width, d, bias=False)

    def _inputs(self, x):
        g = -self.A_log.float().exp() * F.softplus(self.f_proj(x).float() + self.dt_bias)
        v = self.v_proj(x)
        kept = -torch.expm1(2.0 * g)
        shut = kept == 0  # (where the root's slope is infinite, and softplus' slope zero)
        gain = kept.masked_fill(shut, 1.0).sqrt().masked_fill(shut, 0.0)
        return (v * gain).to(v.dtype), g

    def _output(self, h, x):
        heads = (*h.shape[:-1], self.H, self.V)
        return self.o_proj(self.o_norm(h.reshape(heads), self.g_proj(x).reshape(heads)).flatten(-2))

    def forward(self, x, initial_state=None):
        """x [B, T, d] -> (output [B, T, d], final state [B, value_dim])."""
        v, g = self._inputs(x)
        h, state = gated_scan(v, g, initial_state, output_final_state=True)
        return self._output(h, x), state

    @torch.no_grad()
    def step(self, x, state):
        """One token, without gradients: x [B, d], state [B, value_dim] (updated in place) -> [B, d]."""
        v, g = self._inputs(x)
        h, _ = step_gated_scan(v, g, state, out_state=state)
        return self._output(h, x)


class ScaledEmbedding(nn.Embedding):
    """Token embedding times a constant: ``embed_tokens`` on a GPU, torch's
    lookup for what that does not take (a model with another op may run on the
    host, in float64 or under torch.func's transforms)."""

    def __init__(self, num_embeddings: int, dim: int, scale: float = 1.0):
        super().__init__(num_embeddings, dim)
        self.scale = scale

    def forward(self, input_ids):
        if self.weight.is_cuda and self.weight.dtype in _DTYPES and not (
                _is_transformed(self.weight) or _is_transformed(input_ids)):
            return embed_tokens(input_ids, self.weight, self.scale, self.padding_idx)
        y = super().forward(input_ids)
        return y if self.scale == 1.0 else y * self.scale


class NestedGDN2Block(nn.Module):
    """Pre-norm token mixing and channel mixing with residuals
    (modeling_nested_gdn2.py:43-67)."""

    def __init__(self, cfg: ModelConfig, op=None, recurrent=False):
        super().__init__()
        self.attn_norm = RMSNorm(cfg.hidden_size, cfg.norm_eps)
        self.attn = GatedRecurrence(cfg) if recurrent else NestedGDN2Attention(cfg, op)
        self.mlp_norm = RMSNorm(cfg.hidden_size, cfg.norm_eps)
        self.mlp = GatedMLP(cfg.hidden_size, cfg.hidden_ratio, cfg.intermediate_size)

    def forward(self, h):
        a, _ = self.attn(self.attn_norm(h))
        h = h + a
        return h + self.mlp(self.mlp_norm(h))

    @torch.no_grad()
    def step(self, h, state):
        h = h + self.attn.step(self.attn_norm(h), state)
        return h + self.mlp(self.mlp_norm(h))


class NestedGDN2ForCausalLM(nn.Module):
    """Embedding -> blocks -> RMSNorm -> LM head (modeling_nested_gdn2.py:93-160,
    203-268); weights N(0, initializer_range) as ``_init_weights``
    (modeling_nested_gdn2.py:76-90), except the layer's own A_log, dt_bias
    and promotion parameters."""

    def __init__(self, cfg: ModelConfig, op=None):
        super().__init__()
        self.cfg = cfg
        self.embeddings = ScaledEmbedding(cfg.vocab_size, cfg.hidden_size, cfg.embed_scale)
        self.layers = nn.ModuleList(NestedGDN2Block(cfg, op, i in cfg.recurrent_layers)
                                    for i in range(cfg.num_hidden_layers))
        self.norm = RMSNorm(cfg.hidden_size, cfg.norm_eps)
        self.lm_head = nn.Linear(cfg.hidden_size, cfg.vocab_size, bias=False)
        for m in self.modules():
            if isinstance(m, (nn.Linear, nn.Embedding, ShortConvolution)):
                nn.init.normal_(m.weight, mean=0.0, std=cfg.initializer_range)
                if getattr(m, "bias", None) is not None:
                    nn.init.zeros_(m.bias)

    def forward(self, input_ids):
        h = self.embeddings(input_ids)
        for layer in self.layers:
            h = layer(h)
        return self.lm_head(self.norm(h))

    def prefill(self, input_ids):
        """[B, T] ids -> (logits [B, T, V], the layers' states for ``step``);
        for models whose every layer is a GatedRecurrence."""
        self._require_recurrent()
        h, states = self.embeddings(input_ids), []
        for layer in self.layers:
            a, state = layer.attn(layer.attn_norm(h))
            states.append(state)
            h = h + a
            h = h + layer.mlp(layer.mlp_norm(h))
        return self.lm_head(self.norm(h)), states

    @torch.no_grad()
    def step(self, input_ids, states):
        """One decode token for every row: [B] ids -> logits [B, V], without
        gradients; the states (from ``prefill``) are updated in place."""
        self._require_recurrent()
        h = self.embeddings(input_ids)
        for layer, state in zip(self.layers, states, strict=True):
            h = layer.step(h, state)
        return self.lm_head(self.norm(h))

    def _require_recurrent(self):
        if not all(isinstance(layer.attn, GatedRecurrence) for layer in self.layers):
            raise ValueError("token-by-token decoding needs every layer in recurrent_layers: the "
                             "nested layers keep no decode cache here")
