"""Plain 64-bit forms of the decoder-layer operators with the error their
definition allows, element by element, for test_attention.py and
test_gpu_attention.py."""
import torch

F32 = 2.0 ** -24  # half a step of fp32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """half a step below the normal range"""
    return {torch.float16: 2.0 ** -25}.get(dtype, 2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150)


def close(got, want, tol):
    got, want, tol = got.detach().double().cpu(), want.double().cpu(), tol.double().cpu()
    assert got.shape == want.shape, (got.shape, want.shape)
    same = got.isnan() & want.isnan() | (got == want)
    bad = ~(same | ((got - want).abs() <= tol))
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{int(bad.sum())} of {bad.numel()} off; first {i}: {got[i]:.9g} for {want[i]:.9g}, "
                             f"allowed {tol[i]:.3g}; worst {(got - want).abs()[bad].max():.3g}")


def table64(positions, rot, base=10000.0):
    freq = base ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1)


def rotate(x, rows, interleaved, sign=1.0):
    """x [.., heads, dim], rows [.., rot]; also the sum of magnitudes behind each element"""
    half = rows.shape[-1] // 2
    c, s = rows[..., None, :half], sign * rows[..., None, half:]
    i = torch.arange(half) * 2 if interleaved else torch.arange(half)
    j = i + 1 if interleaved else i + half
    y, m = x.clone(), x.abs()
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    m[..., i] = m[..., j] = x[..., i].abs() + x[..., j].abs()
    return y, m


def norm_rope(x, w, pos, rope, eps, interleaved, norm=True):
    """(y, tolerance).  fp32: the row's sum of squares has at most dim roundings (half of it
    after the root), then the root, the weight, the scale and the rotation some more; each is
    relative to the magnitudes that the element is made of.  One rounding to the type."""
    dtype, dim = x.dtype, x.shape[-1]
    x = x.detach().double().cpu()
    pos, rope = pos.long().cpu(), rope.double().cpu()
    there = (pos >= 0) & (pos < rope.shape[0])
    u = x
    if norm:
        u = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        if w is not None:
            u = u * w.detach().double().cpu()
    y, mag = rotate(u, rope[pos.clamp(0, max(rope.shape[0] - 1, 0))], interleaved)
    mask = there[..., None, None]
    y = torch.where(mask, y, torch.zeros(()).double())
    tol = mag * (dim / 2 + 24) * F32 + y.abs() * half_step(dtype) * (1 + 2.0 ** -7) + smallest(dtype)
    return y, tol


def norm_rope_grad(x, w, g, pos, rope, eps, interleaved):
    """(dx, its tolerance, dw, its tolerance)"""
    dtype, dim = x.dtype, x.shape[-1]
    wtype = w.dtype if w is not None else torch.float32
    x, g = x.detach().double().cpu(), g.detach().double().cpu()
    pos, rope = pos.long().cpu(), rope.double().cpu()
    there = ((pos >= 0) & (pos < rope.shape[0]))[..., None, None].double()
    h, hm = rotate(g, rope[pos.clamp(0, max(rope.shape[0] - 1, 0))], interleaved, -1.0)
    h, hm = h * there, hm * there
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    rows = h.numel() // dim
    dw = (h * x * r).flatten(0, -2).sum(0)
    # every term: the rotation, r (dim / 2 + 4 roundings), two products; then at most `rows` additions
    dw_mag = (hm * x.abs() * r).flatten(0, -2).sum(0)
    dw_tol = dw_mag * (dim / 2 + rows + 24) * F32 + dw.abs() * half_step(wtype) * (1 + 2.0 ** -7) + smallest(wtype)
    ww = w.detach().double().cpu() if w is not None else torch.ones(dim, dtype=torch.float64)
    mean = (ww * h * x).mean(-1, keepdim=True)
    mean_mag = (ww.abs() * hm * x.abs()).mean(-1, keepdim=True)
    dx = (r * (ww * h - x * r * r * mean)) * there
    mag = r * (ww.abs() * hm + x.abs() * r * r * mean_mag) * there
    # the mean of dim products and three powers of r
    dx_tol = mag * (dim + 3 * (dim / 2 + 4) + 24) * F32 + dx.abs() * half_step(dtype) * (1 + 2.0 ** -7) + smallest(dtype)
    return dx, dx_tol, dw, dw_tol


def positions_of(cu, lens):
    """(sequence, position) of every token row that belongs to a sequence"""
    out = []
    for b, n in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        out += [(b, n - (t1 - t0) + i) for i in range(t1 - t0)]
    return out


def append(q, k, v, kc, vc, table, cu, lens, rope=None, norm=False, qw=None, kw=None, eps=1e-6, interleaved=False):
    """((q, tolerance), (k_cache, tolerance), (v_cache, 0)): the caches after the call"""
    cu, lens, tab = cu.tolist(), lens.tolist(), table.tolist()
    where = positions_of(cu, lens)
    live = len(where)
    pages, _, page, _ = kc.shape
    pos = torch.tensor([p for _, p in where], dtype=torch.long)
    rows = rope if rope is not None else torch.cat([torch.ones(max(lens + [1]), 4), torch.zeros(max(lens + [1]), 4)], 1)
    kc64, kt = kc.double().cpu().clone(), torch.zeros(kc.shape).double()
    vc64 = vc.double().cpu().clone()
    y, t = norm_rope(k[:live], kw, pos, rows, eps, interleaved, norm)
    for i, (b, p) in enumerate(where):
        if p < 0 or p >= rows.shape[0] or p >= len(tab[b]) * page:
            continue
        at = tab[b][p // page]
        if 0 <= at < pages:
            kc64[at, :, p % page], kt[at, :, p % page] = y[i], t[i]
            vc64[at, :, p % page] = v[i].double().cpu()
    out = None
    if q is not None:
        out64, qt = torch.zeros(q.shape).double(), torch.zeros(q.shape).double()
        out64[:live], qt[:live] = norm_rope(q[:live], qw, pos, rows, eps, interleaved, norm)
        out = (out64, qt)
    return out, (kc64, kt), (vc64, torch.zeros(vc.shape).double())


def attention(q, kc, vc, table, cu, lens, scale=None, causal=True, window=0):
    """(out, tolerance).  A score's sum of dim products has at most dim + 1 roundings (2 F32 each:
    a matrix instruction may cut instead of rounding), the exponent and its scale a few more; a
    relative error e of every weight moves the mean of the values by at most 2 e sum w |v|.  The
    weights are rounded once to the cache's type, their products added in fp32, the result rounded once."""
    dtype = q.dtype
    q64, dim = q.detach().double().cpu(), q.shape[-1]
    scale = dim ** -0.5 if scale is None else scale
    pages, hkv, page, _ = kc.shape
    group = q.shape[1] // hkv
    cu, lens, tab = cu.tolist(), lens.tolist(), table.tolist()
    out, tol = torch.zeros(q.shape).double(), torch.zeros(q.shape).double()
    kc, vc = kc.double().cpu(), vc.double().cpu()
    for b, m in enumerate(lens):
        t0, t1 = cu[b], cu[b + 1]
        n = t1 - t0
        keys = [j for j in range(min(m, len(tab[b]) * page)) if 0 <= tab[b][j // page] < pages]
        if not n or not keys:
            continue
        j = torch.tensor(keys)
        at = torch.tensor([tab[b][x // page] for x in keys])
        pos = torch.arange(m - n, m)[:, None]
        sees = torch.ones(n, len(keys), dtype=torch.bool)
        if causal:
            sees &= j <= pos
        if window:
            sees &= j > pos - window
        for h in range(hkv):
            k, v = kc[at, h, j % page], vc[at, h, j % page]
            for g in range(group):
                x = q64[t0:t1, h * group + g]
                s = (x @ k.t()) * scale
                mag = torch.where(sees, (x.abs() @ k.abs().t()) * scale, torch.zeros(()).double())
                s = s.masked_fill(~sees, float("-inf"))
                top = s.max(1, keepdim=True).values
                w = torch.exp(s - torch.where(top == float("-inf"), torch.zeros(()).double(), top))
                w = torch.where(sees, w, torch.zeros(()).double())
                total = w.sum(1, keepdim=True)
                # a hidden key adds nothing, whatever its value
                vv = torch.where(sees[:, :, None], v[None], torch.zeros(()).double())
                o = torch.where(total == 0, torch.zeros(()).double(), (w[:, :, None] * vv).sum(1) / total)
                a = torch.where(total == 0, torch.zeros(()).double(), (w[:, :, None] * vv.abs()).sum(1) / total)
                e = mag.max(1, keepdim=True).values * ((dim + 1) * 2 + 8) * F32 + 16 * F32
                rel = 2 * e + 2 * (len(keys) + 16) * F32 + (half_step(dtype) if dtype != torch.float32 else 0.0)
                out[t0:t1, h * group + g] = o
                tol[t0:t1, h * group + g] = a * rel * 1.01 + o.abs() * half_step(dtype) + smallest(dtype)
    # (weights below fp16's normal range are off by half a step of 2^-24 each, of a largest weight of 2^7)
    if dtype == torch.float16:
        tol = tol + max(lens + [0]) * 2.0 ** -32 * max(1.0, float(vc[vc.isfinite()].abs().max()) if vc.isfinite().any() else 1.0)
    return out, tol


def batch(new, kv, hq, hkv, dim, page, dtype, device="cpu", seed=0, pad=0, spare=2, layout="heads", stale=float("nan")):
    """A batch whose cache holds its keys and `stale` everywhere else.  layout "tokens": the
    cache's memory is [pages, page, heads, dim] and the tensors are views of it."""
    gen = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in kv]
    pages, width = sum(counts) + spare, max(counts + [1]) + 1
    order = torch.randperm(pages, generator=gen).tolist()
    table, used = torch.full((len(kv), width), -1, dtype=torch.int32), 0
    shape = (pages, hkv, page, dim) if layout == "heads" else (pages, page, hkv, dim)
    kc, vc = torch.full(shape, stale, dtype=dtype), torch.full(shape, stale, dtype=dtype)
    if layout == "tokens":
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    for b, n in enumerate(kv):
        ids = order[used:used + counts[b]]
        used += counts[b]
        table[b, :counts[b]] = torch.tensor(ids, dtype=torch.int32)
        for c in (kc, vc):
            for i, p in enumerate(ids):
                rows = min(page, n - i * page)
                c[p, :, :rows] = torch.randn(hkv, rows, dim, generator=gen).to(dtype)
    tokens = sum(new) + pad
    q = (torch.randn(tokens, hq, dim, generator=gen) * 2).to(dtype)
    k, v = (torch.randn(tokens, hkv, dim, generator=gen).to(dtype) for _ in range(2))
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32)
    lens = torch.tensor(kv, dtype=torch.int32)
    if device != "cpu":  # (.to keeps the views' strides)
        q, k, v, kc, vc, table, cu, lens = (t.to(device) for t in (q, k, v, kc, vc, table, cu, lens))
    return dict(q=q, k=k, v=v, kc=kc, vc=vc, table=table, cu=cu, lens=lens)
