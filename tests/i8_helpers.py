"""Device matrices of the 8-bit layers' and the experts' tests: numpy values in
f32, f16 or bf16 (bf16 as its 16-bit words), rows at any stride and offset, and
the rounding that a result of each type may carry."""
import numpy as np

import zkml_amd as z

TYPES = {"f32": z.F32, "f16": z.F16, "bf16": z.BF16, "i32": z.I32}
# half a unit in the last place of a value of 1 to 2, and of the smallest values
ROUND = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
TINY = {"f32": 2.0**-149, "f16": 2.0**-25, "bf16": 2.0**-134}


def words(a, kind):
    """float64 values rounded to the type: its words (f32/f16: the type itself)."""
    if kind != "bf16":
        return np.asarray(a).astype({"f32": np.float32, "f16": np.float16, "i8": np.int8, "i32": np.int32}[kind])
    f = np.asarray(a, dtype=np.float32)
    u = f.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(f), np.uint16(0x7FC0), r)


def values(w, kind):
    """Words of a type as float64 values."""
    if kind != "bf16":
        return w.astype(np.float64)
    return (w.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


class At:
    """Device memory from an address on (what the front end takes as a buffer)."""

    def __init__(self, buf, offset=0):
        self.buf, self.ptr, self.nbytes = buf, buf.ptr + offset, buf.nbytes - offset


def matrix(ctx, w, ld=None, lead=0, fill=0x55):
    """Uploads the rows of w at stride ld (elements), `lead` elements in; the
    gaps hold `fill` bytes."""
    rows, cols = w.shape
    ld = cols if ld is None else ld
    flat = np.full((lead + max(rows, 1) * ld) * w.itemsize, fill, dtype=np.uint8).view(w.dtype)
    for r in range(rows):
        flat[lead + r * ld:lead + r * ld + cols] = w[r]
    return At(ctx.upload(flat), lead * w.itemsize)


class Result:
    """A result matrix at stride ld, `lead` elements in, its memory filled with
    0xAA bytes; read() gives the rows and checks that the gaps are untouched."""

    def __init__(self, ctx, rows, cols, kind, ld=None, lead=0):
        self.dtype = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i32": np.int32, "i8": np.int8}[kind]
        self.ctx, self.rows, self.cols, self.lead = ctx, rows, cols, lead
        self.ld = cols if ld is None else ld
        self.size = lead + max(rows, 1) * self.ld + 64
        self.all = np.full(self.size * np.dtype(self.dtype).itemsize, 0xAA, dtype=np.uint8).view(self.dtype)
        self.buf = ctx.upload(self.all)
        self.at = At(self.buf, lead * np.dtype(self.dtype).itemsize)

    def read(self):
        got = self.ctx.d2h(self.buf, (self.size,), self.dtype)
        out, want = np.empty((self.rows, self.cols), dtype=self.dtype), self.all.copy()
        for r in range(self.rows):
            s = slice(self.lead + r * self.ld, self.lead + r * self.ld + self.cols)
            out[r] = got[s]
            want[s] = got[s]
        assert got.tobytes() == want.tobytes(), "memory beside the result was written"
        return out
