"""The denoiser with its hidden blocks on microscaled 4-bit operands (`set_gemm_mode("mx4")`): a fast draft of the sampler.

The stack is MLPDiffusion's proj + mlp (`tab_ddpm/modules.py:425-460`).  proj and head stay float32 - they see the table's
columns and the time embedding, and write the noise estimate and the logits - and hold a few per cent of the work; the
hidden blocks' weights are packed once per chain, and every block writes the next one's packed operand itself.  4 bits keep
about one decimal digit per activation: samples differ visibly from the float32 ones, which the split-f16 mode reproduces.
The kernel of a layer, and with it the order of a row's sums, follows from the number of rows (up to 16, up to 64, more): a last
bit of difference there can move a 4-bit rounding of the next layer, so batches of such different sizes can differ in single values.
"""
from . import _lib, ops

_ACT_NAMES = {0: None, 1: "relu", 2: "leaky_relu", 3: "silu"}


class Mx4Stack:
    """weights[l] [d_out, d_in], biases[l], activation codes, as `MLPDiffusion.stack()` returns them."""

    def __init__(self, weights, biases, acts):
        if not (len(weights) == len(biases) == len(acts) >= 2):
            raise _lib.ClavaHipError("Mx4Stack: needs a first and a last layer")
        self.acts = [_ACT_NAMES[int(a)] for a in acts]
        self.biases = [b.detach().float().contiguous() for b in biases]
        self.first, self.last = weights[0].detach().float().contiguous(), weights[-1].detach().float().contiguous()
        self.hidden = [ops.mx4_pack(w.detach()) for w in weights[1:-1]]

    def buffers(self, rows):
        """Operands between the hidden blocks for batches of `rows`: a caller keeps them for as many calls as it makes on one
        stream."""
        return [ops.mx4_empty(rows, w.rows, w.device) for w in self.hidden[:-1]]

    def forward(self, x, rowadd=None, buffers=None):
        """The last layer's output, float32 [B, d_out]; `rowadd` is added to the first layer's pre-activation (`proj(x) + emb`)."""
        h = ops.linear(x, self.first, self.biases[0], act=self.acts[0], rowadd=rowadd)
        if h.shape[0] == 0:
            return ops.linear(h.new_empty(0, self.last.shape[1]), self.last, self.biases[-1])
        buffers = self.buffers(h.shape[0]) if buffers is None else buffers
        for l, w in enumerate(self.hidden, start=1):
            h = ops.linear_mx4(h, w, self.biases[l], act=self.acts[l], out=buffers[l - 1] if l <= len(buffers) else None)
        return ops.linear(h, self.last, self.biases[-1], act=self.acts[-1])
