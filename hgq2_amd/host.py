"""The handful of plain (un-quantized) host-framework names the reference's examples use next to the quantized
layers (reference README.md:57-67: ``keras.Sequential``, ``keras.layers.MaxPooling2D``, ``keras.layers.Flatten``),
on the torch-native layer runtime of ``hgq2_amd.core``.  With ``import hgq2_amd.host as keras`` the README example
runs as written.  Tensors are channels-last, as in Keras."""

from __future__ import annotations

from types import SimpleNamespace

import torch

from . import ops
from .core import Layer, Sequential, get_initializer  # noqa: F401  (Sequential is part of this module's surface)


def _pair(v):
    return (int(v), int(v)) if isinstance(v, int) else tuple(int(t) for t in v)


class _Pooling2D(Layer):
    _mode = 'max'

    def __init__(self, pool_size=(2, 2), strides=None, padding='valid', data_format=None, **kwargs):
        if data_format not in (None, 'channels_last'):
            raise NotImplementedError('pooling: channels_last only')
        super().__init__(**kwargs)
        self.pool_size = _pair(pool_size)
        self.strides = _pair(strides) if strides is not None else self.pool_size
        self.padding = padding.lower()
        if self.padding not in ('valid', 'same'):
            raise ValueError(f'unknown padding {padding!r}')

    def compute_output_shape(self, input_shape):
        out = [input_shape[0]]
        for n, p, s in zip(input_shape[1:3], self.pool_size, self.strides):
            out.append(None if n is None else (-(-n // s) if self.padding == 'same' else (n - p) // s + 1))
        return tuple(out) + (input_shape[3],)

    def call(self, x, training=None):
        return ops.pool2d(x, self.pool_size, self.strides, self.padding, self._mode)

    def get_config(self):
        return {'name': self.name, 'pool_size': self.pool_size, 'strides': self.strides, 'padding': self.padding}

    def host_fn(self, x):
        """The same pooling on a CPU tensor with library routines (for checks against a CPU model)."""
        import torch.nn.functional as F

        t = x.permute(0, 3, 1, 2)
        pads = [0, 0, 0, 0]
        if self.padding == 'same':
            pads = []
            for d in (1, 0):
                n, k, st = t.shape[2 + d], self.pool_size[d], self.strides[d]
                total = max((-(-n // st) - 1) * st + k - n, 0)
                pads += [total // 2, total - total // 2]
        if self._mode == 'max':
            y = F.max_pool2d(F.pad(t, pads, value=float('-inf')), self.pool_size, self.strides)
        else:
            num = F.avg_pool2d(F.pad(t, pads), self.pool_size, self.strides, divisor_override=1)
            cnt = F.avg_pool2d(F.pad(torch.ones_like(t[:1, :1]), pads), self.pool_size, self.strides, divisor_override=1)
            y = num / cnt
        return y.permute(0, 2, 3, 1)


class MaxPooling2D(_Pooling2D):
    _mode = 'max'


class AveragePooling2D(_Pooling2D):
    _mode = 'avg'


class Flatten(Layer):
    def compute_output_shape(self, input_shape):
        n = 1
        for d in input_shape[1:]:
            n *= d
        return (input_shape[0], n)

    def call(self, x, training=None):
        return x.reshape(x.shape[0], -1)

    host_fn = staticmethod(lambda x: x.reshape(x.shape[0], -1))


class GlobalAveragePooling1D(Layer):
    """Mean over the middle axis of a [batch, steps, channels] tensor."""

    def compute_output_shape(self, input_shape):
        return (input_shape[0], input_shape[2])

    def call(self, x, training=None):
        if x.is_cuda and x.dtype == torch.float32 and x.numel():
            return ops.mean_mid(x)
        return torch.mean(x, dim=1)

    host_fn = staticmethod(lambda x: torch.mean(x, dim=1))


class GroupNormalization(Layer):
    """``keras.layers.GroupNormalization`` over the trailing channel axis (same argument names and defaults; ``groups=-1``: each
    channel by itself), with an activation in the same launch.  Full precision, not quantized: what a network trained on small batches
    puts between its layers in the place of a batch normalisation, whose moments such batches do not give.  Variables ``gamma`` and
    ``beta`` are float32; inputs are float32, bfloat16 or float16 GPU tensors ``[batch, ..., channels]``."""

    def __init__(self, groups=32, axis=-1, epsilon=1e-3, center=True, scale=True, beta_initializer='zeros', gamma_initializer='ones',
                 beta_regularizer=None, gamma_regularizer=None, beta_constraint=None, gamma_constraint=None, activation=None, **kwargs):
        super().__init__(**kwargs)
        if activation not in ops.GROUP_ACTIVATIONS:
            raise ValueError(f'GroupNormalization: activation must be one of linear, relu, silu; got {activation!r}')
        if int(groups) < 1 and int(groups) != -1:
            raise ValueError(f'GroupNormalization: groups must be positive, or -1 for as many as channels; got {groups}')
        if not float(epsilon) >= 0:
            raise ValueError('GroupNormalization: epsilon must not be negative')
        self.groups, self.axis, self.epsilon = int(groups), int(axis), float(epsilon)
        self.center, self.scale, self.activation = bool(center), bool(scale), activation
        self.beta_initializer, self.gamma_initializer = get_initializer(beta_initializer), get_initializer(gamma_initializer)
        self.beta_regularizer, self.gamma_regularizer = beta_regularizer, gamma_regularizer
        self.beta_constraint, self.gamma_constraint = beta_constraint, gamma_constraint
        self.gamma = self.beta = None

    def build(self, input_shape):
        input_shape = tuple(input_shape)
        if len(input_shape) < 2 or self.axis % len(input_shape) != len(input_shape) - 1:
            raise NotImplementedError('GroupNormalization: the trailing axis of [batch, ..., channels] only')
        channels = int(input_shape[-1])
        if self.groups == -1:
            self.groups = channels
        if channels % self.groups:
            raise ValueError(f'GroupNormalization: {channels} channels do not fall into {self.groups} groups of one size')
        if self.scale:
            self.gamma = self.add_weight(shape=(channels,), name='gamma', initializer=self.gamma_initializer, regularizer=self.gamma_regularizer,
                                         constraint=self.gamma_constraint)
        if self.center:
            self.beta = self.add_weight(shape=(channels,), name='beta', initializer=self.beta_initializer, regularizer=self.beta_regularizer,
                                        constraint=self.beta_constraint)
        super().build(input_shape)

    def call(self, x, training=None):
        return ops.group_norm(x, self.groups, self.gamma, self.beta, self.epsilon, self.activation)

    def get_config(self):
        return {'name': self.name, 'groups': self.groups, 'axis': self.axis, 'epsilon': self.epsilon, 'center': self.center, 'scale': self.scale,
                'beta_initializer': self.beta_initializer, 'gamma_initializer': self.gamma_initializer, 'beta_regularizer': self.beta_regularizer,
                'gamma_regularizer': self.gamma_regularizer, 'beta_constraint': self.beta_constraint, 'gamma_constraint': self.gamma_constraint,
                'activation': self.activation}

    def host_fn(self, x):
        """The same on a CPU tensor with library routines (for checks against a CPU model)."""
        import torch.nn.functional as F

        vec = [None if t is None else t.detach().to(x.device, x.dtype) for t in (self.gamma, self.beta)]
        y = F.group_norm(x.movedim(-1, 1), self.groups, *vec, self.epsilon).movedim(1, -1)
        return torch.relu(y) if self.activation == 'relu' else F.silu(y) if self.activation in ('silu', 'swish') else y


class RMSNormalization(Layer):
    """``keras.layers.RMSNormalization`` over the trailing axis (variable ``scale``): x / sqrt(mean(x^2) + epsilon) * scale.  Full precision, not
    quantized; inputs are float32, bfloat16 or float16 GPU tensors."""

    def __init__(self, axis=-1, epsilon=1e-6, scale_initializer='ones', **kwargs):
        super().__init__(**kwargs)
        if not float(epsilon) >= 0:
            raise ValueError('RMSNormalization: epsilon must not be negative')
        self.axis, self.epsilon, self.scale_initializer, self.scale = int(axis), float(epsilon), get_initializer(scale_initializer), None

    def build(self, input_shape):
        input_shape = tuple(input_shape)
        if not input_shape or self.axis % len(input_shape) != len(input_shape) - 1:
            raise NotImplementedError('RMSNormalization: the trailing axis only')
        self.scale = self.add_weight(shape=(int(input_shape[-1]),), name='scale', initializer=self.scale_initializer)
        super().build(input_shape)

    def call(self, x, training=None):
        return ops.rms_norm(x, self.scale, self.epsilon)

    def get_config(self):
        return {'name': self.name, 'axis': self.axis, 'epsilon': self.epsilon, 'scale_initializer': self.scale_initializer}


class ResidualBlocks(Layer):
    """A stack of blocks that keep their input's shape (a :class:`QMultiHeadAttention`, a ``Sequential`` of dense layers) on a residual stream, with a norm ahead
    of each and behind each::

        h = norm(x) * gamma_0;   for block k:  x = x + scale * act(gate_k(h)) * norm(block_k(h)) * post_k,   h = norm(x) * gamma_(k + 1)

    and the last h as the output.  Everything between two blocks is one launch each way (:func:`hgq2_amd.ops.residual_norm`); the norms are full precision, the
    blocks quantize their inputs themselves.  ``gates``: a layer (or ``None``) for each block whose output is ``[batch, ..., channels]``, or one row
    for each sample ``[batch, channels]``; ``gate_activation`` ``'sigmoid'`` or ``None``."""

    def __init__(self, blocks, gates=None, gate_activation='sigmoid', scale=1.0, epsilon=1e-6, **kwargs):
        super().__init__(**kwargs)
        blocks = list(blocks)
        if not blocks:
            raise ValueError('ResidualBlocks: at least one block')
        gates = [None] * len(blocks) if gates is None else list(gates)
        if len(gates) != len(blocks):
            raise ValueError(f'ResidualBlocks: {len(blocks)} blocks need as many gates (None for none), got {len(gates)}')
        if gate_activation not in ops.GATE_ACTIVATIONS:
            raise ValueError(f'ResidualBlocks: gate_activation must be one of linear, sigmoid; got {gate_activation!r}')
        if not float(epsilon) >= 0:
            raise ValueError('ResidualBlocks: epsilon must not be negative')
        self.blocks = torch.nn.ModuleList(blocks)
        self.gates = torch.nn.ModuleList([g for g in gates if g is not None])
        self._gated = [g is not None for g in gates]
        self.gate_activation, self.scale, self.epsilon = gate_activation, float(scale), float(epsilon)

    def build(self, input_shape):
        channels = (int(tuple(input_shape)[-1]),)
        for k in range(len(self.blocks) + 1):
            self.add_weight(shape=channels, name=f'gamma_{k}', initializer='ones')
        for k in range(len(self.blocks)):
            self.add_weight(shape=channels, name=f'post_{k}', initializer='ones')
        super().build(input_shape)

    @property
    def same_shape_layers(self):
        return [*self.blocks, *self.gates]

    def call(self, x, training=None):
        var = lambda name: getattr(self, f'_var_{name}')  # noqa: E731
        h = ops.rms_norm(x, var('gamma_0'), self.epsilon)
        gates = iter(self.gates)
        for k, (block, gated) in enumerate(zip(self.blocks, self._gated)):
            gate = next(gates)(h, training=training) if gated else None
            x, h = ops.residual_norm(x, block(h, training=training), var(f'post_{k}'), var(f'gamma_{k + 1}'), gate, self.gate_activation if gated else None, self.scale,
                                     self.epsilon)
        return h

    def get_config(self):
        gates = iter(self.gates)
        return {'name': self.name, 'blocks': list(self.blocks), 'gates': [next(gates) if g else None for g in self._gated], 'gate_activation': self.gate_activation,
                'scale': self.scale, 'epsilon': self.epsilon}


layers = SimpleNamespace(GroupNormalization=GroupNormalization, RMSNormalization=RMSNormalization, MaxPooling2D=MaxPooling2D, AveragePooling2D=AveragePooling2D, Flatten=Flatten,
                         GlobalAveragePooling1D=GlobalAveragePooling1D, Layer=Layer)
