"""MXFP4 and expert routing from their definitions, in 64 bits on the CPU: what
the tests compare the kernels with."""
import numpy as np

GRID = np.array([0, .5, 1, 1.5, 2, 3, 4, 6])
MIDDLES = (GRID[1:] + GRID[:-1]) / 2


def scale_byte(amax):
    """floor(log2 amax) - 2 + 127, not below 0; 255 for NaN and infinities; 0 for 0."""
    amax = np.asarray(amax, np.float64)
    e = np.frexp(np.where(np.isfinite(amax) & (amax > 0), amax, 1.0))[1] - 1
    b = np.where(amax > 0, np.maximum(e - 2 + 127, 0), 0)
    return np.where(np.isfinite(amax), b, 255).astype(np.uint8)


def codes_of(y, byte):
    """Nearest codes of y [.., 32] in blocks with scale bytes [..], ties to the even code."""
    v = y / np.exp2(byte.astype(np.float64) - 127)[..., None]
    a = np.abs(np.where(np.isfinite(v), v, 0.0))
    code = np.zeros(a.shape, np.uint8)
    for i, m in enumerate(MIDDLES):                  # past middle i the code is i + 1; at it the even one of both
        code += ((a > m) | ((a == m) & (i % 2 == 1))).astype(np.uint8)
    code |= np.signbit(np.where(np.isfinite(v), v, 0.0)).astype(np.uint8) << 3
    return np.where(byte[..., None] == 255, 0, code).astype(np.uint8)


def pack(code):
    return code[..., 0::2] | (code[..., 1::2] << 4)


def unpack(packed):
    out = np.empty((*packed.shape[:-1], 2 * packed.shape[-1]), np.uint8)
    out[..., 0::2], out[..., 1::2] = packed & 15, packed >> 4
    return out


def quantize(x):
    """x [.., K] -> (codes uint8 [.., K/2], scale bytes [.., K/32])."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    s = scale_byte(np.abs(b).max(axis=-1))
    return pack(codes_of(b, s).reshape(x.shape)), s


def dequantize(packed, scales):
    c = unpack(np.asarray(packed))
    v = np.where(c & 8, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scales == 255, np.nan, np.exp2(np.asarray(scales, np.float64) - 127))
    return v * np.repeat(s, 32, axis=-1)


def rotation(G):
    h4 = np.array([[1, 1, 1, -1], [1, 1, -1, 1], [1, -1, 1, 1], [-1, 1, 1, 1]], np.float64)
    h = h4
    while h.shape[0] < G:
        h = np.kron(h, h4)
    return h / np.sqrt(G)


def rotate(x, G):
    x = np.asarray(x, np.float64)
    return (x.reshape(-1, G) @ rotation(G)).reshape(x.shape) if G else x


def plan(ids, E):
    """(order, position, offsets) of the stable sort of the slots by expert."""
    flat = np.asarray(ids).reshape(-1)
    used = (flat >= 0) & (flat < E)
    slots = np.nonzero(used)[0]
    slots = slots[np.argsort(flat[slots], kind="stable")]
    order = np.full(flat.shape, -1, np.int32)
    order[:len(slots)] = slots
    position = np.full(flat.shape, -1, np.int32)
    position[slots] = np.arange(len(slots))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[used], minlength=E)[:E])]).astype(np.int32)
    return order, position.reshape(np.shape(ids)), offsets
