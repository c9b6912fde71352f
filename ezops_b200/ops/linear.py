"""A linear layer for any number of rows, with its epilogue: ``out = act(X @ W.T + bias) + residual``.

The projections of the decode operators (ezops/ops/qwen3_dense_decode.py:157-175) as an operator of its own, so that
prompts - hundreds or thousands of rows - go through the same weights.  X [M, K] and W [N, K] are bf16; bias [N] and
residual [M, N] (bf16) are optional; everything behind the product stays in fp32 and is rounded once, to bf16, or not at
all (``out_dtype=torch.float32``, e.g. for scores over a vocabulary).  ``activation``: ``None``, ``"silu"``, ``"gelu"`` (erf form),
``"relu"`` or ``"swiglu"`` - then W is [2N, K] and bias [2N], gate rows before up rows (the layout of ``Wgu``,
ezops/ops/qwen3_dense_decode.py:35), and act is ``silu(gate) * up``.

Rows of X, residual and ``out`` may lie further apart than they are long; ``residual`` may be ``out`` itself (the residual
stream updated in place).  X may have no rows; sizes above 2^30 are refused.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F

from ..registry import get_kernel
from .base_op import Op, rel_frobenius

ACTIVATIONS = {None: 0, "silu": 1, "gelu": 2, "relu": 3, "swiglu": 4}


class LinearOp(Op):
    _params_desc = {
        "rows": "Rows of X that gen_data makes (calls take any number)",
        "out_features": "Columns of the result (N)",
        "in_features": "Columns of X and W (K, a multiple of 8)",
        "bias": "A bias is added to the product",
        "activation": "None, 'silu', 'gelu', 'relu' or 'swiglu' (W then holds gate and up rows)",
        "residual": "A residual is added to the activation",
        "out_dtype": "torch.bfloat16 (default) or torch.float32",
    }
    _rtol = 1e-2

    def __init__(self, rows: int, out_features: int, in_features: int, backend: str = "ref", bias: bool = False, activation=None,
                 residual: bool = False, out_dtype=torch.bfloat16):
        if min(rows, out_features, in_features) < 1:
            raise ValueError("rows, out_features and in_features must be positive")
        if in_features % 8:
            raise ValueError(f"in_features ({in_features}) must be divisible by 8")
        if activation not in ACTIVATIONS:
            raise ValueError(f"activation {activation!r} is none of {list(ACTIVATIONS)}")
        if out_dtype not in (torch.bfloat16, torch.float32):
            raise ValueError(f"out_dtype must be bfloat16 or float32, got {out_dtype}")
        self.rows, self.out_features, self.in_features = rows, out_features, in_features
        self.bias, self.activation, self.residual, self.out_dtype = bool(bias), activation, bool(residual), out_dtype
        self.weight_rows = out_features * (2 if activation == "swiglu" else 1)
        self._backend = backend
        if backend == "ref":
            self._kernel = self._ref_forward
        else:
            self._kernel = get_kernel("linear", backend)(out_features, in_features, bias=self.bias, activation=activation,
                                                         residual=self.residual, out_dtype=out_dtype)

    def forward(self, X, W, bias=None, residual=None, out=None):
        if (bias is None) is self.bias or (residual is None) is self.residual:
            name, expected = ("bias", self.bias) if (bias is None) is self.bias else ("residual", self.residual)
            raise ValueError(f"the operator was made {'with' if expected else 'without'} a {name}")
        return self._kernel(X, W, bias, residual, out)

    def check(self, actual, expected) -> bool:
        return actual.shape == expected.shape and rel_frobenius(actual, expected) < self._rtol

    def gen_data(self, device="cuda"):
        kw = dict(device=device, dtype=torch.bfloat16)
        X = torch.randn(self.rows, self.in_features, **kw)
        W = torch.randn(self.weight_rows, self.in_features, **kw) * self.in_features**-0.5
        bias = torch.randn(self.weight_rows, **kw) if self.bias else None
        residual = torch.randn(self.rows, self.out_features, **kw) if self.residual else None
        return X, W, bias, residual

    def _ref_forward(self, X, W, bias=None, residual=None, out=None):
        z = X.float() @ W.float().T
        if bias is not None:
            z = z + bias.float()
        if self.activation == "swiglu":
            z = F.silu(z[:, : self.out_features]) * z[:, self.out_features :]
        elif self.activation is not None:
            z = getattr(F, self.activation)(z)
        if residual is not None:
            z = z + residual.float()
        z = z.to(self.out_dtype)
        return z if out is None else out.copy_(z)
