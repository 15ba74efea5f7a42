"""Rotary positions: what a model holds of them (ops.rotary applies them).

The reference's positions are a learned table of max_position_embeddings rows (model/model.py:217-245); rotary positions turn the
query / key pairs of every head by angles proportional to the token position instead, need no table row per position, and reach
beyond the trained length by scaling the angles.
"""
import math

import torch

from .._lib import UniterHipError

SCALINGS = ("linear", "ntk", "yarn")


class RotaryPositions(object):
    """Frequencies and layout of rotary positions for heads of `head_dim` elements.

    rotary_dim    leading elements of a head that are turned (even; default: all)
    base          the angle per position of pair i is base ** (-2 i / rotary_dim)
    interleaved   False: pair i is elements (i, rotary_dim / 2 + i); True: (2 i, 2 i + 1)
    scaling       None, or a dict for contexts `factor` times the trained one:
                    {"type": "linear", "factor": f}   every angle divided by f
                    {"type": "ntk", "factor": f}      base multiplied by f ** (rotary_dim / (rotary_dim - 2)): the slowest pair is
                                                      divided by f, the fastest stays
                    {"type": "yarn", "factor": f, "original_max_position": n}
                                                      pairs that make more than beta_fast (32) turns over the n trained positions
                                                      stay, those with fewer than beta_slow (1) are divided by f, a ramp between;
                                                      the result is multiplied by attention_factor (0.1 ln f + 1)

    Not a module and without parameters: `.bfloat16()` of a model must not round the frequencies, which are kept in 64 bits.
    """

    def __init__(self, head_dim, rotary_dim=None, base=10000.0, interleaved=False, scaling=None):
        rot = head_dim if rotary_dim is None else rotary_dim
        if head_dim < 2 or head_dim > 1024:
            raise UniterHipError("rotary: head_dim must be 2 .. 1024, got %r" % (head_dim,))
        if rot < 2 or rot % 2 != 0 or rot > head_dim:
            raise UniterHipError("rotary: rotary_dim must be even and within the head, got %r of %r" % (rot, head_dim))
        if not (base > 0 and math.isfinite(base)):
            raise UniterHipError("rotary: base must be positive, got %r" % (base,))
        self.head_dim, self.rotary_dim, self.base, self.interleaved = int(head_dim), int(rot), float(base), bool(interleaved)
        self.scaling = None if scaling is None else dict(scaling)
        self.multiplier = 1.0
        self.inv_freq = self._frequencies()
        self._turns = {}

    def _frequencies(self):
        """Angle per position of every pair (list of Python floats)."""
        rot, base, s = self.rotary_dim, self.base, self.scaling
        if s is None:
            return [base ** (-2.0 * i / rot) for i in range(rot // 2)]
        kind, factor = s.get("type"), float(s.get("factor", 0.0))
        if kind not in SCALINGS:
            raise UniterHipError("rotary: scaling type must be one of %s, got %r" % (", ".join(SCALINGS), kind))
        known = {"type", "factor"} | ({"original_max_position", "beta_fast", "beta_slow", "attention_factor"} if kind == "yarn" else set())
        # (a scaling made for "yarn" may name the trained length whatever its type)
        odd = set(s) - known - {"original_max_position"}
        if odd:
            raise UniterHipError("rotary: %s scaling has no %s" % (kind, ", ".join(sorted(odd))))
        if not (factor >= 1.0 and math.isfinite(factor)):
            raise UniterHipError("rotary: a scaling factor is 1 or more, got %r" % (s.get("factor"),))
        if kind == "ntk":
            if rot == 2:
                raise UniterHipError("rotary: ntk scaling needs more than one pair")
            base = base * factor ** (rot / (rot - 2.0))
        freq = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
        if kind == "linear":
            return [f / factor for f in freq]
        if kind == "ntk":
            return freq
        trained = s.get("original_max_position")
        if trained is None or trained < 1:
            raise UniterHipError("rotary: yarn scaling needs original_max_position, the trained length")
        if self.base == 1.0:
            raise UniterHipError("rotary: yarn scaling needs a base other than 1")
        fast, slow = float(s.get("beta_fast", 32.0)), float(s.get("beta_slow", 1.0))
        if not fast > slow > 0:
            raise UniterHipError("rotary: yarn scaling needs beta_fast > beta_slow > 0")

        def pair_of(turns):                     # the pair (not whole) that makes so many turns over the trained positions
            return rot * math.log(trained / (turns * 2.0 * math.pi)) / (2.0 * math.log(self.base))

        lo, hi = max(math.floor(pair_of(fast)), 0), min(math.ceil(pair_of(slow)), rot - 1)
        out = []
        for i, f in enumerate(freq):
            stretched = min(1.0, max(0.0, (i - lo) / max(hi - lo, 1e-3)))
            out.append(f / factor * stretched + f * (1.0 - stretched))
        self.multiplier = float(s.get("attention_factor", 0.1 * math.log(factor) + 1.0))
        return out

    def turns(self, device):
        """float64 [rotary_dim / 2] on `device`: turns per position (angle / 2 pi), made once per device.  Not while a graph is being captured:
        the table outlives the graph, and its copy from the host could not be captured."""
        t = self._turns.get(device)
        if t is None:
            device = torch.device(device)
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise UniterHipError("rotary: the first call on %s cannot be captured; call it (or turns(%r)) once before the capture" % (device, str(device)))
            with torch.inference_mode(False):   # (an ordinary tensor whatever the first call runs in: later ones may have gradients)
                t = torch.tensor([f / (2.0 * math.pi) for f in self.inv_freq], dtype=torch.float64, device=device)
            self._turns[device] = t
        return t

    def __deepcopy__(self, memo):
        return self                             # (nothing in it changes: the copies of a layer share it)

    def __getstate__(self):
        return dict(self.__dict__, _turns={})   # device tables are made again where they are needed

    def __repr__(self):
        return "RotaryPositions(head_dim=%d, rotary_dim=%d, base=%g, interleaved=%r, scaling=%r)" % (
            self.head_dim, self.rotary_dim, self.base, self.interleaved, self.scaling)
