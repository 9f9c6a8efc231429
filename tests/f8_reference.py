"""Plain 64-bit arithmetic of the 8-bit operators for their tests: the OCP 8-bit formats, quantisation by blocks of 128,
the scaled product, the root-mean-square norm and its gradient, and storage with pitches, offsets and guard values."""
import numpy as np

from backup_1_amd import capi

BLOCK = 128
LARGEST = {capi.E4M3: 448.0, capi.E5M2: 57344.0}
NP_TYPE = {capi.F32: np.float32, capi.F16: np.float16, capi.BF16: np.uint16}
# half a step relative to the value: what one rounding to the type can be off by
HALF_STEP = {capi.F32: 2.0 ** -24, capi.F16: 2.0 ** -11, capi.BF16: 2.0 ** -8}
TYPE_NAMES = {capi.F32: "f32", capi.F16: "f16", capi.BF16: "bf16"}


def decode_table(fmt):
    """The value of each of the 256 codes, from the formats' definition."""
    ebits, mbits, bias = (4, 3, 7) if fmt == capi.E4M3 else (5, 2, 15)
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> mbits) & ((1 << ebits) - 1), c & ((1 << mbits) - 1)
        v = m * 2.0 ** (1 - bias - mbits) if e == 0 else (1 + m / (1 << mbits)) * 2.0 ** (e - bias)
        if fmt == capi.E4M3 and (c & 0x7F) == 0x7F:
            v = np.nan
        if fmt == capi.E5M2 and e == 31:
            v = np.inf if m == 0 else np.nan
        out[c] = -v if c & 0x80 else v
    return out


TABLE = {f: decode_table(f) for f in (capi.E4M3, capi.E5M2)}


def encode(v, fmt):
    """Codes of the nearest values, ties to the even code; finite input within the format's range."""
    grid = TABLE[fmt][:128]
    grid = grid[np.isfinite(grid)]                              # ascending, code = index
    a = np.abs(np.asarray(v, np.float64))
    hi = np.clip(np.searchsorted(grid, a), 0, grid.size - 1)
    lo = np.maximum(hi - 1, 0)
    up, down = grid[hi] - a, a - grid[lo]
    code = np.where((down < up) | ((down == up) & (lo % 2 == 0)), lo, hi)
    code = np.where(grid[hi] <= a, hi, code)
    return (code | np.where(np.signbit(v), 0x80, 0)).astype(np.uint8)


def bf16_round(v):
    """float32 -> the nearest bfloat16, as its bits (finite values)."""
    u = np.ascontiguousarray(v, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def to_type(v, kind):
    """float32 values as the type's storage."""
    v = np.asarray(v, np.float32)
    return bf16_round(v) if kind == capi.BF16 else v.astype(NP_TYPE[kind])


def from_type(a, kind):
    """Storage -> float64."""
    if kind == capi.BF16:
        return (a.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    return a.astype(np.float64)


def scale_values(s):
    """Stored scales (fp32, or biased exponents) -> float64."""
    if s.dtype == np.uint8:
        return np.where(s == 255, np.nan, 2.0 ** (s.astype(np.float64) - 127))
    return s.astype(np.float64)


def block_amax(x, block_rows):
    M, K = x.shape
    p = np.zeros((-(-M // block_rows) * block_rows, -(-K // BLOCK) * BLOCK))
    p[:M, :K] = np.abs(x)
    return p.reshape(-1, block_rows, p.shape[1] // BLOCK, BLOCK).max((1, 3))


def spread(s, M, K, block_rows):
    """[column block][row block] scales -> one for each element."""
    return s.T[np.arange(M) // block_rows][:, np.arange(K) // BLOCK]


def quantize(x, fmt, scale_type, block_rows):
    """x float32-valued (M, K) -> codes (M, K), stored scales [ceil(K/128)][row blocks]: the definition, bit for bit."""
    amax = np.maximum(block_amax(x, block_rows), 2.0 ** -100).astype(np.float32)
    if scale_type == capi.SCALE_F32:
        s = (amax.astype(np.float64) / LARGEST[fmt]).astype(np.float32)
        factor = (1.0 / s.astype(np.float64)).astype(np.float32)
        stored = s
    else:
        e = np.ceil(np.log2(amax.astype(np.float64) / LARGEST[fmt])).astype(int)
        e = np.where(LARGEST[fmt] * 2.0 ** (e - 1.0) >= amax, e - 1, e)
        e = np.where(LARGEST[fmt] * 2.0 ** e < amax, e + 1, e)
        factor = (2.0 ** -e.astype(np.float64)).astype(np.float32)
        stored = (e + 127).astype(np.uint8)
    scaled = x.astype(np.float32) * spread(factor.T, x.shape[0], x.shape[1], block_rows)
    return encode(scaled, fmt), np.ascontiguousarray(stored.T)


def dequantize(codes, fmt, s, block_rows):
    return TABLE[fmt][codes] * spread(scale_values(s), codes.shape[0], codes.shape[1], block_rows)


class Pitched:
    """A rows x cols matrix on the device: a pitch, an offset of `lead` elements from the allocation's start, and a guard
    value everywhere else, which `result` checks."""

    def __init__(self, arr, pitch=None, lead=0, guard=None, tail=64):
        arr = np.ascontiguousarray(arr)
        if arr.ndim == 1:
            arr = arr[None]
        self.rows, self.cols = arr.shape
        self.ld = pitch or self.cols
        self.lead, self.dtype = lead, arr.dtype
        guard = {1: 0x7F, 2: 0x7FC1, 4: 0x7FC00001}[arr.itemsize] if guard is None else guard          # NaNs of every type
        self.store = np.full(lead + self.rows * self.ld + tail, guard, {1: np.uint8, 2: np.uint16, 4: np.uint32}[arr.itemsize])
        bits = arr.view(self.store.dtype)
        self.body(self.store)[:] = bits
        self.buf = capi.DeviceBuffer.from_numpy(self.store)
        self.ptr = self.buf.ptr + lead * arr.itemsize

    def body(self, store):
        return store[self.lead:self.lead + self.rows * self.ld].reshape(self.rows, self.ld)[:, :self.cols]

    @classmethod
    def empty(cls, rows, cols, dtype, **kw):
        return cls(np.full((rows, cols), 0x55, np.dtype(dtype)) if np.dtype(dtype).kind != "f" else np.full((rows, cols), -77.0, dtype), **kw)

    def result(self):
        got = self.buf.download(self.store.shape, self.store.dtype)
        out = self.body(got).copy()
        inside = np.zeros(self.store.shape, bool)
        self.body(inside)[:] = True
        assert np.array_equal(got[~inside], self.store[~inside]), "wrote outside the matrix"
        return out.view(self.dtype)
