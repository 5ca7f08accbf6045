"""How a categorical column's value is chosen from its class probabilities: temperature, top-k, top-p, min-p.

The reference draws from the plain posterior (`log_sample_categorical`, `tab_ddpm/gaussian_multinomial_diffsuion.py:506-516`);
a `CategoryChoice` narrows the draw of the chain's last step, or of a single `p_sample_index`, to the likelier classes.
"""
import math
import sys

import torch

_FIELDS = ("temperature", "top_k", "top_p", "min_p")


class CategoryChoice:
    """Each parameter is a number for all columns, or a sequence with one for every categorical column (0 / 1.0 / 0.0 leave
    top_k / top_p / min_p off; a sequence's temperature, top_p and min_p are rounded to float32).  Definitions:
    `ops.sample_categories`."""
    __slots__ = _FIELDS

    def __init__(self, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        checks = {"temperature": lambda v: 0.0 <= v <= sys.float_info.max, "top_k": lambda v: 0 <= v < math.inf and v == int(v),
                  "top_p": lambda v: 0.0 <= v <= 1.0, "min_p": lambda v: 0.0 <= v <= 1.0}
        for name, value in zip(_FIELDS, (temperature, top_k, top_p, min_p)):
            each = list(value) if isinstance(value, (list, tuple)) else [value]
            for v in each:
                if isinstance(v, bool) or not isinstance(v, (int, float)) or not checks[name](v):
                    raise ValueError(f"CategoryChoice: {name} = {v!r}")
            setattr(self, name, tuple(each) if isinstance(value, (list, tuple)) else value)

    def arguments(self, features, device):
        """Keyword arguments of `ops.sample_categories` for a table of that many categorical columns."""
        out = {}
        for name in _FIELDS:
            v = getattr(self, name)
            if name == "top_k":                                  # (more than a table has classes, in 32 bits)
                v = tuple(min(int(k), 2 ** 31 - 1) for k in v) if isinstance(v, tuple) else min(int(v), 2 ** 31 - 1)
            if isinstance(v, tuple):
                if len(v) != features:
                    raise ValueError(f"CategoryChoice: {len(v)} values of {name} for {features} categorical columns")
                v = torch.tensor(v, device=device, dtype=torch.int32 if name == "top_k" else torch.float32)
            out[name] = v
        return out

    def __repr__(self):
        return "CategoryChoice(" + ", ".join(f"{n}={getattr(self, n)!r}" for n in _FIELDS) + ")"
