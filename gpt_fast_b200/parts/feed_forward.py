"""Feed-forwards.  SwiGLU (gpt-fast model.py:219-227): w2(silu(w1 x) * w3 x); `Dense`: down(act(up x)).

w1 (gate) and w3 (up) are stored as one matrix whose rows alternate gate, up,
so that one product yields both and its epilogue applies silu(gate) * up
before anything is written; the second product adds into the residual."""
import torch

from .. import ops
from ..weights.loader import ParamSpec
from . import register_feed_forward
from .residual import as_residual


@register_feed_forward("swiglu")
class SwiGLU:
    def __init__(self, dim: int, hidden: int, dtype: torch.dtype):
        self.dim, self.hidden, self.dtype = dim, hidden, dtype
        self.w13 = self.w2 = None
        self.int8_weights = False

    def param_specs(self):
        return {"w1": ParamSpec((self.hidden, self.dim)), "w3": ParamSpec((self.hidden, self.dim)),
                "w2": ParamSpec((self.dim, self.hidden))}

    def load(self, tensors):
        self.w13 = torch.stack([tensors["w1"], tensors["w3"]], dim=1).reshape(2 * self.hidden, self.dim).contiguous()
        self.w2 = tensors["w2"]

    def quantize(self):
        """Both matrices as 8-bit integers with a scale per output."""
        self.w13, self.w2, self.int8_weights = ops.quantize_rows(self.w13), ops.quantize_rows(self.w2), True

    def export(self):
        """The parameters as `load` received them (gate and up rows taken apart again)."""
        w = self.w13.view(self.hidden, 2, self.dim)
        return {"w1": w[:, 0], "w3": w[:, 1], "w2": self.w2}

    def forward(self, h, residual):
        act = torch.empty(h.shape[0], self.hidden, dtype=self.dtype, device=h.device)
        ops.linear(h, self.w13, act, mode="swiglu")
        as_residual(residual).add_linear(act, self.w2)


@register_feed_forward("dense")
class Dense:
    """Two products with a unary activation between them: down(act(up x)).  activation: 'gelu' (the exact one,
    0.5 z (1 + erf(z / sqrt 2))), 'gelu_tanh', 'silu' or 'relu2' (the square of max(z, 0)); it is applied in the first
    product's epilogue."""

    ACTIVATIONS = ("gelu", "gelu_tanh", "silu", "relu2")

    def __init__(self, dim: int, hidden: int, dtype: torch.dtype, activation: str = "gelu"):
        if activation not in self.ACTIVATIONS:
            raise ValueError(f"unknown activation '{activation}'; known: {self.ACTIVATIONS}")
        self.dim, self.hidden, self.dtype, self.activation = dim, hidden, dtype, activation
        self.up = self.down = None
        self.int8_weights = False

    def param_specs(self):
        return {"up": ParamSpec((self.hidden, self.dim)), "down": ParamSpec((self.dim, self.hidden))}

    def load(self, tensors):
        self.up, self.down = tensors["up"], tensors["down"]

    def quantize(self):
        """Both matrices as 8-bit integers with a scale per output."""
        self.up, self.down, self.int8_weights = ops.quantize_rows(self.up), ops.quantize_rows(self.down), True

    def export(self):
        return {"up": self.up, "down": self.down}

    def forward(self, h, residual):
        act = torch.empty(h.shape[0], self.hidden, dtype=self.dtype, device=h.device)
        ops.linear(h, self.up, act, mode=self.activation)
        as_residual(residual).add_linear(act, self.down)
