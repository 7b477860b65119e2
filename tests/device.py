"""Device arrays of a test: uploaded from numpy, read back by address, freed together."""
import numpy as np


class Arrays:
    def __init__(self, ctx):
        self.ctx, self.held = ctx, {}

    def up(self, a) -> int:
        a = np.ascontiguousarray(a)
        p = self.ctx.upload(a if a.size else np.zeros(1, np.uint8))
        self.held[p] = (a.shape, a.dtype)
        return p

    def down(self, p: int) -> np.ndarray:
        self.ctx.synchronize()
        shape, dtype = self.held[p]
        return self.ctx.download(p, shape, dtype)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.ctx.synchronize()
        for p in self.held:
            self.ctx.free(p)


NP = {"f32": np.float32, "f16": np.float16}


def guarded(a: np.ndarray, before: int, after: int, fill) -> np.ndarray:
    """`a` flattened between guard elements of `fill`."""
    return np.concatenate([np.full(before, fill, a.dtype), a.reshape(-1), np.full(after, fill, a.dtype)])
