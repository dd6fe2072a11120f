"""Layer factories and the gated residual block, API-compatible with the reference's
``wavenet_vocoder.modules`` (modules.py:13-169).  ``ResidualConv1dGLU.incremental_forward`` runs as one
HIP kernel per step (``wnv_glu_step``); the batch ``forward`` is ordinary torch ops (parity oracle and
likelihood scoring, not the hot path).

``ResidualRecurrentGLU`` is its recurrent counterpart, which the reference has not: the same contract, a gated linear recurrence
(``recurrence.gated_recurrence``) in place of the dilated convolution, trained by the scan and its backward pass and served by its
step, with 4-bit projections on request."""
from __future__ import annotations

import math

import torch
from torch import nn
from torch.nn import functional as F

from . import conv
from .engine import GluLayer, Q4Linear, require_gpu_tensor
from .recurrence import gated_recurrence, gated_recurrence_step

__all__ = ["Conv1d", "Embedding", "Conv1d1x1", "ResidualConv1dGLU", "ResidualRecurrentGLU"]


def Conv1d(in_channels, out_channels, kernel_size, dropout=0, **kwargs):
    """He-initialised conv (the reference adds weight norm on top, modules.py:13-18; with g initialised
    to ||v|| the effective weight is the same tensor, and this package keeps weights fused)."""
    m = conv.Conv1d(in_channels, out_channels, kernel_size, **kwargs)
    nn.init.kaiming_normal_(m.weight, nonlinearity="relu")
    if m.bias is not None:
        nn.init.constant_(m.bias, 0)
    return m


def Embedding(num_embeddings, embedding_dim, padding_idx, std=0.01):
    m = nn.Embedding(num_embeddings, embedding_dim, padding_idx=padding_idx)
    m.weight.data.normal_(0, std)
    return m


def Conv1d1x1(in_channels, out_channels, bias=True):
    return Conv1d(in_channels, out_channels, kernel_size=1, padding=0, dilation=1, bias=bias)


class ResidualConv1dGLU(nn.Module):
    """Dilated causal conv -> (+ local / global conditioning 1x1) -> tanh * sigmoid -> skip 1x1 and
    residual 1x1.  Constructor signature of reference modules.py:71-75."""

    def __init__(self, residual_channels, gate_channels, kernel_size, skip_out_channels=None,
                 cin_channels=-1, gin_channels=-1, dropout=1 - 0.95, padding=None, dilation=1,
                 causal=True, bias=True, *args, **kwargs):
        super().__init__()
        self.dropout = dropout
        if skip_out_channels is None:
            skip_out_channels = residual_channels
        if padding is None:
            padding = (kernel_size - 1) * dilation if causal else (kernel_size - 1) // 2 * dilation
        self.causal = causal
        self.conv = Conv1d(residual_channels, gate_channels, kernel_size, padding=padding,
                           dilation=dilation, bias=bias, *args, **kwargs)
        self.conv1x1c = Conv1d1x1(cin_channels, gate_channels, bias=False) if cin_channels > 0 else None
        self.conv1x1g = Conv1d1x1(gin_channels, gate_channels, bias=False) if gin_channels > 0 else None
        half = gate_channels // 2
        self.conv1x1_out = Conv1d1x1(half, residual_channels, bias=bias)
        self.conv1x1_skip = Conv1d1x1(half, skip_out_channels, bias=bias)
        self._geom = dict(residual_channels=residual_channels, gate_channels=gate_channels,
                          kernel_size=kernel_size, skip_out_channels=skip_out_channels,
                          cin_channels=cin_channels, gin_channels=gin_channels, dilation=dilation, bias=bias)
        self._glu = None
        self._glu_key = None

    # -- batch path (torch ops) ------------------------------------------------------------------
    def forward(self, x, c=None, g=None):
        """x (B,R,T), c (B,cin,T), g (B,gin,T) -> (x', s); reference modules.py:109-110,127-163."""
        residual = x
        x = F.dropout(x, p=self.dropout, training=self.training)
        x = self.conv(x)
        if self.causal:
            x = x[:, :, :residual.size(-1)]
        a, b = x.split(x.size(1) // 2, dim=1)
        if c is not None:
            assert self.conv1x1c is not None
            ca, cb = self.conv1x1c(c).split(x.size(1) // 2, dim=1)
            a, b = a + ca, b + cb
        if g is not None:
            assert self.conv1x1g is not None
            ga, gb = self.conv1x1g(g).split(x.size(1) // 2, dim=1)
            a, b = a + ga, b + gb
        z = torch.tanh(a) * torch.sigmoid(b)
        s = self.conv1x1_skip(z)
        o = self.conv1x1_out(z)
        return (o + residual) * math.sqrt(0.5), s

    # -- incremental path (HIP) ------------------------------------------------------------------
    def _engine(self) -> GluLayer:
        params = [p for p in self.parameters()]
        require_gpu_tensor(params[0], "ResidualConv1dGLU parameters")
        key = tuple((p.device, p.data_ptr(), p._version) for p in params)
        if self._glu is None or self._glu_key != key:
            self._glu = GluLayer(device=params[0].device, **self._geom)
            self._glu.load_weights({k: v for k, v in self.state_dict().items()})
            self._glu_key = key
        return self._glu

    def incremental_forward(self, x, c=None, g=None):
        """x (B,1,R), c (B,1,cin), g (B,1,gin) -> (x' (B,1,R), s (B,1,K)); reference modules.py:112-113."""
        if self.training:
            raise RuntimeError('incremental_forward only supports eval mode')     # conv.py:19-20
        if c is not None:
            assert self.conv1x1c is not None                                      # modules.py:142
        if g is not None:
            assert self.conv1x1g is not None                                      # modules.py:149
        B = x.size(0)
        xo, so = self._engine().step(x[:, -1, :], None if c is None else c[:, -1, :],
                                     None if g is None else g[:, -1, :])
        return xo.view(B, 1, -1), so.view(B, 1, -1)

    def invalidate_engine(self):
        """Drop the packed weights of the layer-level engine (see WaveNet.invalidate_engine)."""
        self._glu, self._glu_key = None, None

    def clear_buffer(self):
        if self._glu is not None:
            self._glu.reset()
        for m in (self.conv, self.conv1x1_out, self.conv1x1_skip, self.conv1x1c, self.conv1x1g):
            if m is not None:
                m.clear_buffer()


class ResidualRecurrentGLU(nn.Module):
    """1x1 projection to the gates (+ local / global conditioning 1x1) -> gated linear recurrence -> skip 1x1 and residual 1x1; the
    contract of ``ResidualConv1dGLU`` with one state of ``gate_channels // 2`` numbers an utterance for a past of any length.

    z = conv1x1_in(x) + conv1x1c(c) + conv1x1g(g) = (f | v | o), y = ``gated_recurrence(z)``, s = conv1x1_skip(y),
    x' = (conv1x1_out(y) + x) sqrt(1/2).  Runs on the GPU only, in both forms."""

    def __init__(self, residual_channels, gate_channels, skip_out_channels=None, cin_channels=-1, gin_channels=-1,
                 dropout=1 - 0.95, bias=True):
        super().__init__()
        self.dropout = dropout
        if skip_out_channels is None:
            skip_out_channels = residual_channels
        half = gate_channels // 2
        self.half = half
        self.conv1x1_in = Conv1d1x1(residual_channels, 3 * half, bias=bias)
        self.conv1x1c = Conv1d1x1(cin_channels, 3 * half, bias=False) if cin_channels > 0 else None
        self.conv1x1g = Conv1d1x1(gin_channels, 3 * half, bias=False) if gin_channels > 0 else None
        self.conv1x1_out = Conv1d1x1(half, residual_channels, bias=bias)
        self.conv1x1_skip = Conv1d1x1(half, skip_out_channels, bias=bias)
        self._state = None
        self._q4_group = None
        self._q4_gates = self._q4_heads = None      # apart: in a copy of the module each is None
        self._q4_key = None

    # -- batch path: training and scoring ----------------------------------------------------------
    def forward(self, x, c=None, g=None, lengths=None, seg_start=None):
        """x (B,R,T), c (B,cin,T), g (B,gin,T) -> (x', s), of the projections' type; ``lengths`` and ``seg_start`` as in
        ``recurrence.gated_recurrence``."""
        residual = x
        x = F.dropout(x, p=self.dropout, training=self.training)
        z = self._project(self.conv1x1_in, x)
        if c is not None:
            assert self.conv1x1c is not None
            z = z + self._project(self.conv1x1c, c)
        if g is not None:
            assert self.conv1x1g is not None
            z = z + self._project(self.conv1x1g, g)
        y, _ = gated_recurrence(z, lengths=lengths, seg_start=seg_start)
        s = self._project(self.conv1x1_skip, y.transpose(1, 2)).transpose(1, 2)
        o = self._project(self.conv1x1_out, y.transpose(1, 2)).transpose(1, 2)
        return (o + residual) * math.sqrt(0.5), s

    @staticmethod
    def _project(m, x):
        """A 1x1 convolution of (B, C, T), channels last as the recurrence reads it: (B, T, C')."""
        return F.linear(x.transpose(1, 2), m.weight.squeeze(-1), m.bias)

    # -- incremental path (HIP) ------------------------------------------------------------------
    def quantize_(self, group_size=64):
        """The steps run on weights of 4 bits from now on (``engine.Q4Linear``), rounded from the module's own at the next step, and
        again after those change; ``group_size=None``: back to float32."""
        self._q4_group = group_size
        self.invalidate_engine()
        return self

    def _engine(self):
        params = list(self.parameters())
        require_gpu_tensor(params[0], "ResidualRecurrentGLU parameters")
        key = tuple((p.device, p.data_ptr(), p._version) for p in params)
        if self._q4_gates is None or self._q4_key != key:
            def layer(convs, dim, **kw):
                w = torch.cat([m.weight.detach().squeeze(-1).float() for m in convs if m is not None], dim)
                biases = [m.bias.detach().float() for m in convs if m is not None and m.bias is not None]
                q = Q4Linear(w.shape[1], w.shape[0], w.device, group_size=self._q4_group, **kw)
                q.set_weights(w, torch.cat(biases) if biases else None)
                return q
            # what adds up shares its inputs side by side, what shares an input its outputs
            self._q4_gates = layer((self.conv1x1_in, self.conv1x1c, self.conv1x1g), 1, gates=3)
            self._q4_heads = layer((self.conv1x1_out, self.conv1x1_skip), 0)
            self._q4_key = key
        return self._q4_gates, self._q4_heads

    def incremental_forward(self, x, c=None, g=None):
        """x (B,1,R), c (B,1,cin), g (B,1,gin) -> (x' (B,1,R), s (B,1,K))."""
        if self.training:
            raise RuntimeError('incremental_forward only supports eval mode')     # conv.py:19-20
        for given, m in ((c, self.conv1x1c), (g, self.conv1x1g)):
            if given is not None:
                assert m is not None
        B = x.size(0)
        if self._state is None:
            require_gpu_tensor(x, "x")
            self._state = torch.zeros(B, self.half, device=x.device)
        elif self._state.shape[0] != B:
            raise ValueError(f"batch size changed from {self._state.shape[0]} to {B} without clear_buffer()")
        with torch.no_grad():
            x = x[:, -1, :].float()
            if self._q4_group is None:
                z = self.conv1x1_in.incremental_forward(x[:, None])
                if c is not None:
                    z = z + self.conv1x1c.incremental_forward(c)
                if g is not None:
                    z = z + self.conv1x1g.incremental_forward(g)
                y = gated_recurrence_step(z[:, 0], self._state)[:, None]
                o, s = self.conv1x1_out.incremental_forward(y)[:, 0], self.conv1x1_skip.incremental_forward(y)[:, 0]
            else:
                gates, heads = self._engine()
                parts = [x]
                for given, m in ((c, self.conv1x1c), (g, self.conv1x1g)):
                    if m is not None:
                        parts.append(x.new_zeros(B, m.in_channels) if given is None else given[:, -1, :].float())
                y = gates.recurrence_step(torch.cat(parts, 1) if len(parts) > 1 else x, self._state)
                o, s = heads.step(y).split((x.shape[1], self.conv1x1_skip.out_channels), 1)
            return ((o + x) * math.sqrt(0.5)).view(B, 1, -1), s.reshape(B, 1, -1)

    def invalidate_engine(self):
        """Drop the packed weights (see WaveNet.invalidate_engine)."""
        self._q4_gates = self._q4_heads = self._q4_key = None
        for m in (self.conv1x1_in, self.conv1x1_out, self.conv1x1_skip, self.conv1x1c, self.conv1x1g):
            if m is not None:
                m.invalidate_engine()

    def clear_buffer(self):
        self._state = None
        for m in (self.conv1x1_in, self.conv1x1_out, self.conv1x1_skip, self.conv1x1c, self.conv1x1g):
            if m is not None:
                m.clear_buffer()
