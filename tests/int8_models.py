"""The plain model with its layers' matrices in 8 bits: every product of a layer reads a weight whose rows, and an operand whose rows, stand for 8-bit
integers times a scale, by the definition (scale = max |row| / 127, halves to even)."""
import torch

import plain_llama as P
from helpers import TOLERANCE

# How far an engine's logits may be from the plain model's, in parts of the largest (helpers.errors). A value that stands next to a border between two integers
# falls to the other side where a sum was rounded otherwise, in float32 too, and that one step does not stay alone. With s the deviation of an operand's
# values, their largest about 4 s and a step D = 4 s / 127 = 3.1 % of s: a step moves the results of its row, sums of k products with k = 64 to 256, by D / sqrt(k) =
# 0.2 to 0.4 % of their deviation. Each value of the next operand is then off by d = 0.3 % of s, which takes it over a border in d / D = a tenth of all cases,
# by D: 3.1 % * sqrt(0.1) = 1 % of s. From there on it is as if the row's operands had been rounded with other borders, D / sqrt(12) * sqrt(2) = 1.3 % of s an
# operand, and the rows that attend to it follow. The bfloat16 model has the same from its first operand on: what it rounds moves a value by up to 2^-9 of it.
# Both are so allowed 1.3 % for each of four operands a layer where the bfloat16 model with plain weights is allowed its roundings of 2^-9 / sqrt(3) * 2 = 0.23 %
# (six a layer): sqrt(4 / 6) * 1.3 / 0.23 = 4.6, five times as much.
LIMITS = {name: 5 * value for name, value in TOLERANCE["bfloat16"].items()}


def in_8_bits(rows):
    """What the rows stand for when they are brought to 8 bits, in 64 bits (the integers and scales are float32's)."""
    rows = rows.to(torch.float32)
    most = rows.abs().amax(-1, keepdim=True)
    scales = most / torch.full_like(most, 127.0)
    values = torch.where(scales > 0, rows / scales, torch.zeros_like(rows)).round().clamp(-127, 127)
    return values.double() * scales.double()


class PlainInt8Model(P.PlainModel):
    """weights: those of the folder; as_bound: the type in which the engine holds a matrix before it is brought to 8 bits."""

    def prepare(self, as_bound):
        self.exact = {name: in_8_bits(tensor.to(as_bound)) for name, tensor in self.weights.items() if tensor.dim() == 2 and ".layers." in name}
        return self

    def block(self, layer, x, positions, tail=0):
        plain = P.linear
        by_identity = {id(self.weights[name]): exact for name, exact in self.exact.items()}
        P.linear = lambda rows, weight: (in_8_bits(rows) @ by_identity[id(weight)].t()).to(rows.dtype)
        try:
            return super().block(layer, x, positions, tail)
        finally:
            P.linear = plain
