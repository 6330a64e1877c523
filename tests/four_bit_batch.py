"""A batch of sequences over a 4-bit cache, for the attention tests: the rows of
``attend_oracle.Batch`` packed as e2m1 codes with e4m3 scales, NaN scales where no
query looks."""
from __future__ import annotations

import torch

import attend_oracle
import token_oracle


class Batch(attend_oracle.Batch):
    def __init__(self, *, heads, group, dim, dtype, factors=(1.0, 1.0), **kw):
        layout = kw.pop("layout", "nhd")
        super().__init__(heads=heads, group=group, dim=dim, dtype=dtype, cache=torch.float32, **kw)
        self.layout = layout
        self.scales = {} if factors == (1.0, 1.0) else dict(key_scale=factors[0], value_scale=factors[1])
        self.rows = []
        for name in ("key", "value"):
            plane = getattr(self, name)
            rows = token_oracle.pack(plane.flatten(0, 1), heads, dim)
            n = heads * dim * 9 // 16
            rows[:, n:] = 0xff  # what is not used may hold anything
            rows = rows.view(*plane.shape[:2], -1)
            self.rows.append(rows)
            setattr(self, name, token_oracle.values(rows, heads, dim))

    def expect(self, p_eps, **kw):
        """As before, with what weights far below the largest may be off.  They are fp16, held times 2^7 of a maximum that
        lags by up to 2^8: a step of 2^-24 there, half of it rounded away, over a sum of 2^7 at least, is 2^-32 of each
        value that a query sees.  It shows here because 4-bit values are often 0, where a tiny weight of another token is
        all of a result."""
        rows, (out, lse, bound, lse_bound) = super().expect(p_eps, **kw)
        top = self.value.nan_to_num().abs().max().item() * self.scales.get("value_scale", 1.0)
        return rows, (out, lse, bound + max(self.lens) * top * 2.0 ** -32, lse_bound)

    def on(self, dev):
        if self.layout == "merged":
            both = torch.stack(self.rows, 2).to(dev)
            return both[:, :, 0], both[:, :, 1]
        if self.layout == "apart":  # tokens 64 bytes further apart than they are long, blocks in another order
            wide = [torch.full((r.shape[1], r.shape[0], r.shape[2] + 64), 0xff, dtype=torch.uint8) for r in self.rows]
            for w, r in zip(wide, self.rows):
                w[:, :, :r.shape[2]] = r.transpose(0, 1)
            return tuple(w.to(dev).transpose(0, 1)[:, :, :r.shape[2]] for w, r in zip(wide, self.rows))
        return tuple(r.to(dev) for r in self.rows)
