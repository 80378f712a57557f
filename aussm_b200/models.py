"""The callers of the scan operators: AUSSM / Mamba blocks and the two model
families the benchmark configurations use, written against this package's
operators.

These are re-statements of the reference's PyTorch modules with the SAME
parameter names and shapes, so that a reference checkpoint's ``state_dict``
loads unchanged (ai-modules/wavesAI/model/aussm.py: ``SSMTS`` :100-227,
``SSMSequenceClassifier`` :382-536, ``ResidualBlock`` :681-714, ``MambaBlock``
:717-805, ``SSMauBlock`` :808-902, ``RMSNorm`` :905-916).  Only the scan calls
differ: ``SSMauBlock`` calls ``aussm_b200.ops.ssm_adaptive_interface`` and
``MambaBlock`` calls ``aussm_b200.s6.selective_scan_fn`` (the reference imports
the latter from the third-party package mamba-ssm); and the ``nn.Linear``
layers are ``aussm_b200.linear.SplitLinear`` (same parameters; the float32
products run on the tensor cores through the library's split GEMM).

``GatedDeltaBlock`` (layer kind ``g``) has no counterpart in the reference: a
mixer with a matrix state next to the two with vector states, in the same
residual blocks and models.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from . import delta, ops, rotary, s6, stages
from .linear import SplitLinear, split_linear

__all__ = ["RMSNorm", "SSMauBlock", "MambaBlock", "GatedDeltaBlock", "ResidualBlock", "SSMTS", "SSMSequenceClassifier"]


class RMSNorm(nn.Module):
    def __init__(self, d_model: int, eps: float = 1e-5):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(d_model))

    def forward(self, x):
        if torch.jit.is_scripting():
            return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + self.eps) * self.weight
        return stages.rms_norm(x, self.weight, self.eps)


def _causal_depthwise_conv(conv: nn.Conv1d, x_bld: torch.Tensor) -> torch.Tensor:
    """(b, l, d) -> (b, l, d): the block's depthwise convolution, cut back to l steps (causal)."""
    l = x_bld.shape[1]
    return conv(x_bld.transpose(1, 2))[:, :, :l].transpose(1, 2)


class SSMauBlock(nn.Module):
    """AUSSM mixer: in_proj -> depthwise conv -> adaptive unitary scan -> out_proj (aussm.py:808-902)."""

    def __init__(self, d_model: int, d_state: int, dt_rank=None, d_conv: int = 4, conv_bias: bool = True,
                 bias: bool = False, conv_1d: bool = True):
        super().__init__()
        self.d_model, self.d_state, self.use_conv = d_model, d_state, conv_1d
        dt_rank = d_state if dt_rank in (None, "auto") else dt_rank
        self.in_proj = SplitLinear(d_model, 2 * d_model, bias=bias)
        self.conv1d = nn.Conv1d(d_model, d_model, kernel_size=d_conv, groups=d_model, padding=d_conv - 1,
                                bias=conv_bias)
        self.out_proj = SplitLinear(d_model, d_model, bias=bias)
        self.x_proj = SplitLinear(d_model, dt_rank, bias=False)
        self.dt_proj = SplitLinear(dt_rank, d_model, bias=True)
        self.D = nn.Parameter(torch.ones(d_model))
        self.C = nn.Parameter(torch.randn(d_state, dtype=torch.complex64))
        self.B = nn.Parameter(torch.randn(d_state, dtype=torch.complex64))
        self.xA_proj = SplitLinear(d_model, d_model * d_state, bias=True)
        with torch.no_grad():
            self.xA_proj.bias.uniform_(-math.pi, math.pi)

    def _operator_parameters(self):
        # xA_proj's rows are ordered (state, channel): weight (n*d, d) -> x[i][j][r], bias -> x_bias[i][j]
        d, n = self.d_model, self.d_state
        x_param = self.xA_proj.weight.view(n, d, d).transpose(0, 1).contiguous() * (1.0 / math.sqrt(d))
        x_bias = self.xA_proj.bias.view(n, d).transpose(0, 1).contiguous()
        return x_param, x_bias

    def forward(self, x):
        if x.is_cuda and x.dtype == torch.float32 and self.conv1d.kernel_size[0] <= 4:
            return self._forward_channel_major(x)
        # The reference's order of operations, token-major with transposes (aussm.py:849-902).  CUDA tensors
        # take the channel-major path below; this one is what the module-glue test pins against the reference's
        # own class on the CPU (with the oracle's scan substituted for the operator).
        b, l, d = x.shape
        xs, z = self.in_proj(x).split([d, d], dim=-1)
        if self.use_conv:
            xs = _causal_depthwise_conv(self.conv1d, xs)
        # the step size: the reference adds dt_proj's bias a second time before the softplus (aussm.py:878-880)
        dt = F.softplus(self.dt_proj(self.x_proj(xs)) + self.dt_proj.bias)
        x_param, x_bias = self._operator_parameters()
        y = ops.ssm_adaptive_interface(u=xs.transpose(1, 2).contiguous(), dt=dt.transpose(1, 2).contiguous(),
                                       x=x_param, x_bias=x_bias, B=self.B, C=self.C, D=self.D.float(),
                                       z=z.transpose(1, 2).contiguous(), unitary=True)
        return self.out_proj(y.transpose(1, 2))

    def _forward_channel_major(self, x):
        """The same block with every stage producing (b, d, l) directly: the linear layers write channel-major
        results, the convolution with its bias and the step size (softplus with the doubled bias) are one
        pass each, and no transposing copy exists on either side of the operator."""
        d = self.d_model
        w_in, b_in = self.in_proj.weight, self.in_proj.bias
        xs = stages.project_tokens(w_in[:d], x)                      # (b, d, l)
        z = stages.project_tokens(w_in[d:], x)
        if b_in is not None:
            xs = xs + b_in[:d, None]
            z = z + b_in[d:, None]
        u = stages.causal_conv_bias(xs, self.conv1d.weight, self.conv1d.bias) if self.use_conv else xs
        low = stages.project_channels(self.x_proj.weight, u)         # (b, rank, l)
        pre = stages.project_channels(self.dt_proj.weight, low)      # (b, d, l), dt_proj without its bias
        dt = stages.softplus_bias(pre, self.dt_proj.bias, 2.0)       # the bias enters twice (aussm.py:878-880)
        x_param, x_bias = self._operator_parameters()
        y = ops.ssm_adaptive_interface(u=u, dt=dt, x=x_param, x_bias=x_bias, B=self.B, C=self.C, D=self.D.float(),
                                       z=z, unitary=True)
        return stages.project_back(self.out_proj.weight, y, self.out_proj.bias)


class MambaBlock(nn.Module):
    """Mamba (S6) mixer (aussm.py:717-805)."""

    def __init__(self, d_model: int, d_state: int = 16, expand: int = 2, dt_rank=None, d_conv: int = 4,
                 conv_bias: bool = True, bias: bool = False):
        super().__init__()
        self.d_model, self.d_state = d_model, d_state
        self.d_inner = int(expand * d_model)
        self.dt_rank = math.ceil(d_model / 16) if dt_rank in (None, "auto") else dt_rank
        self.in_proj = SplitLinear(d_model, 2 * self.d_inner, bias=bias)
        self.conv1d = nn.Conv1d(self.d_inner, self.d_inner, kernel_size=d_conv, groups=self.d_inner,
                                padding=d_conv - 1, bias=conv_bias)
        self.out_proj = SplitLinear(self.d_inner, d_model, bias=bias)
        self.x_proj = SplitLinear(self.d_inner, self.dt_rank + 2 * d_state, bias=False)
        self.dt_proj = SplitLinear(self.dt_rank, self.d_inner, bias=True)
        self.D = nn.Parameter(torch.ones(self.d_inner))
        self.A_log = nn.Parameter(torch.log(torch.arange(1, d_state + 1, dtype=torch.float32)).repeat(self.d_inner, 1))
        self.A_log._no_weight_decay = True

    def forward(self, x):
        if x.is_cuda and x.dtype == torch.float32 and self.conv1d.kernel_size[0] <= 4:
            return self._forward_channel_major(x)
        # the reference's token-major order of operations (aussm.py:749-805); see SSMauBlock.forward
        di, n = self.d_inner, self.d_state
        xs, z = self.in_proj(x).split([di, di], dim=-1)
        xs = _causal_depthwise_conv(self.conv1d, xs)
        dt, Bm, Cm = self.x_proj(xs).split([self.dt_rank, n, n], dim=-1)
        # dt_proj is applied with its bias, and the bias goes in once more as delta_bias (aussm.py:786-799)
        y = s6.selective_scan_fn(F.silu(xs).transpose(1, 2).contiguous(), self.dt_proj(dt).transpose(1, 2).contiguous(),
                                 (-torch.exp(self.A_log.float())).contiguous(), Bm.transpose(1, 2).contiguous(),
                                 Cm.transpose(1, 2).contiguous(), self.D.float().contiguous(),
                                 z=z.transpose(1, 2).contiguous(), delta_bias=self.dt_proj.bias.float(),
                                 delta_softplus=True)
        return self.out_proj(y.transpose(1, 2))


    def _forward_channel_major(self, x):
        """Channel-major form of the block (see SSMauBlock._forward_channel_major)."""
        di, n, r = self.d_inner, self.d_state, self.dt_rank
        w_in, b_in = self.in_proj.weight, self.in_proj.bias
        xs = stages.project_tokens(w_in[:di], x)
        z = stages.project_tokens(w_in[di:], x)
        if b_in is not None:
            xs = xs + b_in[:di, None]
            z = z + b_in[di:, None]
        xs = stages.causal_conv_bias(xs, self.conv1d.weight, self.conv1d.bias)
        low = stages.project_channels(self.x_proj.weight, xs)       # (b, rank + 2n, l): dt, B, C rows
        dt = stages.project_channels(self.dt_proj.weight, low[:, :r].contiguous())
        # dt_proj is applied with its bias, and the bias goes in once more as delta_bias (aussm.py:786-799): both here
        y = s6.selective_scan_fn(F.silu(xs), dt, (-torch.exp(self.A_log.float())).contiguous(),
                                 low[:, r:r + n].contiguous(), low[:, r + n:].contiguous(),
                                 self.D.float().contiguous(), z=z, delta_bias=2.0 * self.dt_proj.bias.float(),
                                 delta_softplus=True)
        return stages.project_back(self.out_proj.weight, y, self.out_proj.bias)


# Up to so many new tokens go one at a time: 16 tokens of 1, 16 and 256 sequences, 8 heads of 128, take 25, 39 and 261 us
# that way and 49, 35 and 341 us in chunks; 32 tokens 30, 72 and 488 against 49, 35 and 352 us.
STEPS = 16


class GatedDeltaBlock(nn.Module):
    """Gated delta rule mixer: in_proj -> depthwise conv, SiLU -> queries and keys to unit length (and rotated) -> gated
    delta rule -> norm of every head, gate -> out_proj.

    ``n_heads`` heads of ``d_model / n_heads`` keys and values (default: the fewest of at most 128); ``rotary_dim`` > 0
    rotates that many elements of every query and key by position.  ``forward`` takes whole sequences (b, l, d),
    ``step`` the next tokens of each (one, or a prompt) with the ``cache`` of ``init_cache``, for serving."""

    def __init__(self, d_model: int, n_heads: int = None, d_conv: int = 4, conv_bias: bool = True, bias: bool = False,
                 rotary_dim: int = 0, rotary_base: float = 10000.0):
        super().__init__()
        if n_heads is None:
            n_heads = next(h for h in range(1, d_model + 1) if d_model % h == 0 and d_model // h <= delta.MAX_KEY)
        if d_model % n_heads or d_model // n_heads > delta.MAX_KEY:
            raise ValueError(f"{n_heads} heads do not cut {d_model} channels into heads of at most {delta.MAX_KEY}")
        if rotary_dim < 0 or rotary_dim % 2 or rotary_dim > d_model // n_heads:
            raise ValueError(f"rotary_dim must be even and at most the head's {d_model // n_heads}, got {rotary_dim}")
        self.d_model, self.n_heads, self.d_head = d_model, n_heads, d_model // n_heads
        self.rotary_dim, self.rotary_base = rotary_dim, rotary_base
        self.in_proj = SplitLinear(d_model, 4 * d_model, bias=bias)          # q, k, v and the gate z
        self.gate_proj = SplitLinear(d_model, 2 * n_heads, bias=False)       # decay and step size of every head
        self.conv1d = nn.Conv1d(3 * d_model, 3 * d_model, kernel_size=d_conv, groups=3 * d_model, padding=d_conv - 1, bias=conv_bias)
        self.out_proj = SplitLinear(d_model, d_model, bias=bias)
        self.norm = RMSNorm(self.d_head)
        self.A_log = nn.Parameter(torch.log(torch.empty(n_heads).uniform_(1, 16)))
        # softplus(dt_bias) spread over 0.001 .. 0.1: heads that remember a thousand steps and heads that remember ten
        dt = torch.exp(torch.empty(n_heads).uniform_(math.log(0.001), math.log(0.1)))
        self.dt_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.A_log._no_weight_decay = True
        self._angles = {}

    def _frequencies(self, device):
        if not self.rotary_dim:
            return None
        if device not in self._angles:       # float64 whatever type the module is cast to
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("GatedDeltaBlock: call the block once before it is captured into a graph")
            with torch.inference_mode(False):    # kept for training too, whoever calls first ..
                kept = rotary.rotary_frequencies(self.rotary_dim, self.rotary_base, device=device)[0]
            if device.type == "cuda":            # .. and for every stream
                torch.cuda.current_stream(device).synchronize()
            self._angles[device] = kept
        return self._angles[device]

    def _inputs(self, x, conv, positions):
        """q, k, v, g, beta from the tokens x and their convolved q, k, v channels (b, l, 3 d)."""
        b, l, _ = x.shape
        q, k, v = F.silu(conv).view(b, l, 3, self.n_heads, self.d_head).unbind(2)
        q, k = rotary.qk_norm_rotate(q, k, self._frequencies(x.device), positions, norm="l2")
        a, beta = self.gate_proj(x).float().split([self.n_heads, self.n_heads], dim=-1)
        g = -torch.exp(self.A_log.float()) * F.softplus(a + self.dt_bias.float())
        return q, k, v, g, torch.sigmoid(beta)

    def _output(self, o, z):
        b, l = o.shape[:2]
        return self.out_proj((self.norm(o) * F.silu(z.view(b, l, self.n_heads, self.d_head))).reshape(b, l, self.d_model))

    def forward(self, x):
        d = self.d_model
        if x.is_cuda and x.dtype == torch.float32 and self.conv1d.kernel_size[0] <= 4 and not torch.is_autocast_enabled("cuda"):
            w, bias = self.in_proj.weight, self.in_proj.bias
            xs = stages.project_tokens(w[:3 * d], x)                         # (b, 3d, l): the convolution's layout
            xs = xs if bias is None else xs + bias[:3 * d, None]
            z = split_linear(x, w[3 * d:], None if bias is None else bias[3 * d:])
            conv = stages.causal_conv_bias(xs, self.conv1d.weight, self.conv1d.bias).transpose(1, 2).contiguous()
        else:
            xs, z = self.in_proj(x).split([3 * d, d], dim=-1)
            conv = _causal_depthwise_conv(self.conv1d, xs).contiguous()
        q, k, v, g, beta = self._inputs(x, conv, None)
        return self._output(delta.gated_delta_rule(q, k, v, g, beta), z)

    def init_cache(self, batch: int, device=None, dtype=None):
        """What ``step`` carries from token to token: the state (float32), the convolution's last inputs, the position (all
        on the device: a captured step moves on when it is replayed).  Device and type default to the block's."""
        h, w = self.n_heads, self.d_head
        device = self.conv1d.weight.device if device is None else device
        dtype = self.conv1d.weight.dtype if dtype is None else dtype
        return dict(state=torch.zeros(batch, h, w, w, device=device, dtype=torch.float32),
                    position=torch.zeros(1, device=device, dtype=torch.int64),
                    conv=torch.zeros(batch, self.conv1d.kernel_size[0] - 1, 3 * self.d_model, device=device, dtype=dtype))

    @torch.no_grad()
    def step(self, x, cache):
        """The next token of every sequence, or the next ones (a prompt): x (b, l, d) -> (b, l, d); ``cache`` is updated in
        place."""
        d, l, w, bias = self.d_model, x.shape[1], self.conv1d.weight, self.conv1d.bias
        xs, z = self.in_proj(x).split([3 * d, d], dim=-1)
        window = torch.cat((cache["conv"], xs), 1)                           # (b, k - 1 + l, 3d)
        if l == 1:
            conv = torch.einsum("bkc,ck->bc", window, w[:, 0])[:, None]
            conv = conv if bias is None else conv + bias
        elif x.is_cuda and window.dtype == w.dtype == torch.float32 and w.shape[2] <= 4:
            conv = stages.causal_conv_bias(window.transpose(1, 2), w, bias).transpose(1, 2)[:, w.shape[2] - 1:]
        else:
            conv = _causal_depthwise_conv(self.conv1d, window)[:, w.shape[2] - 1:]
        cache["conv"].copy_(window[:, l:])
        positions = cache["position"] + torch.arange(l, device=x.device) if self.rotary_dim else None
        q, k, v, g, beta = self._inputs(x, conv.contiguous(), positions)
        cache["position"] += l
        if l <= STEPS:
            return self._output(delta.gated_delta_step(q, k, v, g, beta, cache["state"]), z)
        o, state = delta.gated_delta_rule(q, k, v, g, beta, initial_state=cache["state"], return_final_state=True)
        cache["state"].copy_(state)
        return self._output(o, z)


def _has_hooks(m: nn.Module) -> bool:
    from torch.nn.modules import module as hooks
    return bool(type(m) is not RMSNorm or "forward" in m.__dict__ or m._forward_hooks or m._forward_pre_hooks
                or m._backward_hooks or m._backward_pre_hooks or hooks._global_forward_hooks
                or hooks._global_forward_pre_hooks or hooks._global_backward_hooks
                or hooks._global_backward_pre_hooks)


class ResidualBlock(nn.Module):
    """x + mixer(norm(x))."""

    def __init__(self, mixer: nn.Module, d_model: int):
        super().__init__()
        self.mixer = mixer
        self.norm = RMSNorm(d_model)

    def forward(self, x):
        if _has_hooks(self.norm):              # somebody watches the norm: call it as a module
            return self.mixer(self.norm(x)) + x
        normed, residual = stages.rms_norm_residual(x, self.norm.weight, self.norm.eps)
        return self.mixer(normed) + residual


def _build_layers(layers: str, d_model, d_state, mamba_expand, dt_rank, d_conv, conv_bias, bias, ssmau_conv_1d):
    blocks = []
    for kind in layers.replace(" ", "").split("|"):
        if kind == "a":
            mixer = SSMauBlock(d_model, d_state, dt_rank, d_conv, conv_bias, bias, ssmau_conv_1d)
        elif kind == "m":
            mixer = MambaBlock(d_model, d_state, mamba_expand, dt_rank, d_conv, conv_bias, bias)
        elif kind == "g":
            mixer = GatedDeltaBlock(d_model, d_conv=d_conv, conv_bias=conv_bias, bias=bias)
        else:
            raise NotImplementedError(f'Layer type "{kind}" not recognized')
        blocks.append(ResidualBlock(mixer, d_model))
    return nn.ModuleList(blocks)


class SSMTS(nn.Module):
    """Time-series model: Linear embedding -> 'a|m|g|...' residual blocks -> RMSNorm -> Linear head, per step."""

    def __init__(self, d_model: int, input_dim: int, output_dim: int, layers: str = "m|a", d_state: int = 16,
                 mamba_expand: int = 2, dt_rank="auto", d_conv: int = 4, conv_bias: bool = True, bias: bool = False,
                 ssmau_conv_1d: bool = True):
        super().__init__()
        self.embedding = SplitLinear(input_dim, d_model)
        self.layers = _build_layers(layers, d_model, d_state, mamba_expand, dt_rank, d_conv, conv_bias, bias,
                                    ssmau_conv_1d)
        self.norm_f = RMSNorm(d_model)
        self.output = SplitLinear(d_model, output_dim, bias=False)

    def forward(self, x):
        x = self.embedding(x)
        for layer in self.layers:
            x = layer(x)
        return self.output(self.norm_f(x))


class SSMSequenceClassifier(nn.Module):
    """Token classifier: Embedding -> blocks -> pool over time ("meanpool" or "last") -> RMSNorm -> Linear."""

    def __init__(self, d_model: int, vocab_size: int, output_dim: int, layers: str = "m|a", d_state: int = 16,
                 mamba_expand: int = 2, dt_rank="auto", d_conv: int = 4, conv_bias: bool = True, bias: bool = False,
                 mode: str = "meanpool", ssmau_conv_1d: bool = True):
        super().__init__()
        self.meanpool = "meanpool" in mode
        self.embedding = nn.Embedding(vocab_size, d_model)
        self.layers = _build_layers(layers, d_model, d_state, mamba_expand, dt_rank, d_conv, conv_bias, bias,
                                    ssmau_conv_1d)
        self.norm_f = RMSNorm(d_model)
        self.output = SplitLinear(d_model, output_dim, bias=False)

    def forward(self, input_ids, lengths=None):
        x = self.embedding(input_ids)
        for layer in self.layers:
            x = layer(x)
        if lengths is not None:
            idx = torch.arange(x.shape[1], device=x.device)[None, :]
            if self.meanpool:
                mask = (idx < lengths[:, None]).to(x.dtype)[..., None]
                x = (x * mask).sum(1) / lengths[:, None].to(x.dtype)
            else:
                x = x[torch.arange(x.shape[0], device=x.device), lengths - 1]
        else:
            x = x.mean(1) if self.meanpool else x[:, -1]
        return self.output(self.norm_f(x))
