"""Plain 64-bit forms of the expert-layer operators, for the tests."""
import torch

U = 2.0 ** -24                      # half a step of float32, relative
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the smallest step: what rounding to a subnormal may add."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def randn(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol, what=""):
    """|got - want| <= tol elementwise; NaN and infinities equal."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    same = torch.where(torch.isnan(want), torch.isnan(got), got == want)
    assert bool(same[~fine].all()), f"{what}: not the same infinities and NaN"
    err = torch.where(fine, (got - want).abs(), 0.0)
    bad = fine & ~(err <= tol)
    if bool(bad.any()):
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off; at {i} "
                             f"{got[i].item()!r}, want {want[i].item()!r}, tolerance "
                             f"{torch.broadcast_to(torch.as_tensor(tol), want.shape)[i].item():g}")


def padded(t, lead, fill=float("nan")):
    """t's values in rows with `lead` more columns, which hold `fill`."""
    wide = torch.full((t.shape[0], t.shape[1] + lead), fill, dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def offsets_of(sizes):
    out = [0]
    for s in sizes:
        out.append(out[-1] + s)
    return torch.tensor(out, dtype=torch.int32, device="cuda")


def epilogue(v, name):
    if name == "relu":
        return v.clamp_min(0)
    return torch.where(v < 0, torch.expm1(v), v) if name == "elu" else v


def grouped(x, w, offsets, rows=None, bias=None, epi="none", transpose=False):
    """(y, bound) of grouped_matmul in 64 bits: bound is the sum of |x||w| and
    |bias|, of which a float32 sum is off by (k + 2) 2^-24 at most.  Rows in
    no group are NaN."""
    x, w = x.double(), w.double()
    if transpose:
        w = w.transpose(1, 2)
    if rows is not None:
        r = rows.long()
        inside = (r >= 0) & (r < x.shape[0])
        x = torch.where(inside[:, None], x[r.clamp(0, x.shape[0] - 1)], 0.0)
    off = offsets.tolist()
    y = torch.full((x.shape[0], w.shape[2]), float("nan"), dtype=torch.float64, device=x.device)
    size = torch.zeros_like(y)
    for g, (a, b) in enumerate(zip(off, off[1:])):
        if b <= a:
            continue
        y[a:b] = x[a:b] @ w[g]
        size[a:b] = x[a:b].abs() @ w[g].abs()
        if bias is not None:
            y[a:b] += bias[g].double()
            size[a:b] += bias[g].double().abs()
    return epilogue(y, epi), size


def wgrad(x, dy, offsets, rows=None):
    """(dw, its bound, dbias, its bound) in 64 bits."""
    x, dy = x.double(), dy.double()
    if rows is not None:
        r = rows.long()
        inside = (r >= 0) & (r < x.shape[0])
        x = torch.where(inside[:, None], x[r.clamp(0, x.shape[0] - 1)], 0.0)
    off = offsets.tolist()
    out = [[], [], [], []]
    for a, b in zip(off, off[1:]):
        p, d = x[a:b], dy[a:b]
        for o, v in zip(out, (p.t() @ d, p.abs().t() @ d.abs(), d.sum(0), d.abs().sum(0))):
            o.append(v)
    return [torch.stack(o) for o in out]


def e4m3(x):
    """(values that x stands for, q, scale [rows, blocks]) of rows quantised in
    blocks of 128, the definition's roundings in float32."""
    rows, k = x.shape
    kb = -(-k // 128)
    full = torch.zeros(rows, kb * 128, device=x.device)
    full[:, :k] = x.float()
    blocks = full.view(rows, kb, 128)
    scale = (blocks.abs().amax(2) * (1 / 448)).clamp_min(2.0 ** -126)
    q = (blocks / scale[:, :, None]).to(torch.float8_e4m3fn)
    value = (q.double() * scale.double()[:, :, None]).view(rows, -1)[:, :k]
    return value, q.view(rows, -1), scale
