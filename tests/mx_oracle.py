"""Microscaled storage in 64 bits, from its definition (CPU, float64)."""
import torch

BLOCK, GROUP = 32, 128
GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
DT = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
# unit roundoff of a result rounded once to the type
UNIT = {"fp32": 2.0 ** -24, "fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def _exponent(top):
    """floor(log2(top)) of positive doubles."""
    m, e = torch.frexp(top)
    return e.double() - 1


def quantise(x, fmt):
    """x [rows, n] float64 -> (codes, scale bytes), both padded to whole groups of 128:
    codes [rows, groups * 128] int64 (E2M1 code or signed byte), bytes [rows, groups * 4]."""
    rows, n = x.shape
    width = -(-n // GROUP) * GROUP
    b = torch.zeros((rows, width), dtype=torch.float64)
    b[:, :n] = x
    b = b.view(rows, -1, BLOCK)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    top = torch.where(bad, torch.ones_like(top), top)
    e = _exponent(torch.where(top == 0, torch.ones_like(top), top))
    # the largest magnitude rounded (half up) to one mantissa bit, or to six
    limit = 1.75 if fmt == "fp4" else 1 + 127 / 128
    e = e + (top / 2.0 ** e >= limit).double() - (2 if fmt == "fp4" else 0)
    e = e.clamp(-126, 125 if fmt == "fp4" else 127)  # (elements saturate rather than read as infinity)
    v = torch.where(bad[..., None], torch.zeros_like(b), b) / (2.0 ** e)[..., None]
    if fmt == "fp4":
        # nearest of the eight magnitudes; of two as near, the one of even code
        d = (v.abs()[..., None] - GRID).abs()
        lo = d.argmin(-1)
        hi = 7 - d.flip(-1).argmin(-1)
        code = torch.where(lo % 2 == 0, lo, hi) + 8 * ((v < 0) & (hi + lo > 0)).long()
    else:
        code = torch.round(v * 64).clamp(-127, 127).long()
    byte = torch.where(bad, 255, torch.where(top == 0, 0, (e + 127).long()))
    code = torch.where(((byte == 0) | (byte == 255))[..., None], 0, code)
    return code.view(rows, width), byte


def values(code, byte, n, fmt):
    rows = code.shape[0]
    v = torch.cat([GRID, -GRID])[code] if fmt == "fp4" else code.double() / 64
    v = v.view(rows, -1, BLOCK) * (2.0 ** (byte.double() - 127))[..., None]
    v = torch.where((byte == 255)[..., None], torch.full_like(v, float("nan")), v)
    return v.view(rows, -1)[:, :n]


def pack(x, fmt):
    """The package's layout of quantise(x): (codes, scales) tensors."""
    code, byte = quantise(x.double(), fmt)
    rows, n = x.shape
    scales = byte.view(rows, -1, 4).transpose(0, 1).to(torch.uint8).contiguous()
    if fmt == "fp4":
        c = code.view(rows, -1, 2)
        return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8).contiguous(), scales
    return code[:, :-(-n // BLOCK) * BLOCK].to(torch.int8).contiguous(), scales


def quantised(x, fmt):
    code, byte = quantise(x.double(), fmt)
    return values(code, byte, x.shape[1], fmt)


def f(name, x):
    k = (2 / torch.pi) ** 0.5
    return {"identity": lambda: x, "relu": lambda: torch.relu(x), "tanh": lambda: torch.tanh(x),
            "sigmoid": lambda: torch.sigmoid(x), "silu": lambda: x * torch.sigmoid(x),
            "gelu": lambda: 0.5 * x * (1 + torch.tanh(k * (x + 0.044715 * x ** 3)))}[name]()


def df(name, x):
    k = (2 / torch.pi) ** 0.5
    s, t = torch.sigmoid(x), torch.tanh(k * (x + 0.044715 * x ** 3))
    return {"identity": lambda: torch.ones_like(x), "relu": lambda: (x > 0).double(),
            "tanh": lambda: 1 - torch.tanh(x) ** 2, "sigmoid": lambda: s * (1 - s),
            "silu": lambda: s * (1 + x * (1 - s)),
            "gelu": lambda: 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * k * (1 + 3 * 0.044715 * x * x)}[name]()


def product_bound(a, b, n):
    """Bound on the error of sum_k a b in fp32, whatever the order: every one of
    the n additions off by at most 2^-23 of the magnitudes summed."""
    return (n + 8) * 2.0 ** -23 * (a.abs() @ b.abs())
