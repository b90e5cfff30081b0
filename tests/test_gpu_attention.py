"""torch.ops.nnsx.qk_norm_rope / paged_append / paged_attention: the CDNA4 kernels
(csrc/kernels/attn.hip, rope.hip) against 64-bit forms of their definitions."""
import pytest
import torch

import attn_oracle as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module")
def ops(nns):
    return torch.ops.nnsx


def attend(ops, s, **kw):
    return ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], **kw)


def check(ops, s, causal=True, window=0, scale=None):
    got = attend(ops, s, causal=causal, window=window, scale=scale)
    ref.close(got, *ref.attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], scale, causal, window))
    return got


# ------------------------------------------------------------- attention ----

# new tokens, lengths, query heads, kv heads, head dim, page
BATCHES = [
    ([1], [1], 1, 1, 8, 4), ([1], [0], 2, 1, 64, 16), ([0], [5], 2, 1, 64, 16), ([5], [3], 2, 2, 64, 16),
    ([1], [33], 8, 2, 128, 16), ([1, 1, 1], [31, 32, 129], 4, 1, 64, 32), ([2, 9], [70, 9], 4, 4, 32, 1),
    ([3, 0, 1, 6], [10, 4, 33, 6], 6, 2, 24, 3), ([40, 1], [40, 200], 14, 2, 72, 24), ([17], [300], 33, 1, 128, 100),
    ([70, 5], [70, 261], 4, 4, 160, 16), ([9], [200], 3, 3, 256, 64), ([1] * 5, [1, 64, 65, 257, 500], 16, 1, 128, 64),
    ([130], [130], 3, 1, 96, 16), ([1], [700], 5, 5, 80, 256), ([33, 300], [333, 300], 2, 2, 64, 48),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,kv,hq,hkv,dim,page", BATCHES)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 20), (False, 0), (False, 7)])
def test_paged_attention(ops, dtype, new, kv, hq, hkv, dim, page, causal, window):
    s = ref.batch(new, kv, hq, hkv, dim, page, dtype, "cuda", pad=2, seed=len(new) + dim)
    got = check(ops, s, causal, window)
    assert (got[sum(new):] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_paged_attention_long(ops, dtype, dim):
    """one token behind a long context: the keys are split over workgroups and joined"""
    check(ops, ref.batch([1, 2], [5000, 3333], 4, 2, dim, 16, dtype, "cuda"))
    check(ops, ref.batch([1, 4], [5000, 700], 4, 1, dim, 24, dtype, "cuda"), window=1111)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("hq,hkv,dim,page", [(4, 4, 64, 16), (8, 2, 128, 64), (5, 1, 128, 24), (2, 1, 96, 16), (2, 2, 256, 32)])
def test_paged_attention_prompt(ops, dtype, hq, hkv, dim, page):
    """hundreds of new tokens, some behind an earlier part"""
    check(ops, ref.batch([515, 130, 1, 259], [515, 700, 30, 260], hq, hkv, dim, page, dtype, "cuda", pad=1))


def test_paged_attention_many_sequences(ops):
    """more sequences than a workgroup has threads, a third of them without new tokens"""
    new = [(i % 3) for i in range(700)]
    kv = [n + (i * 7) % 90 for i, n in enumerate(new)]
    check(ops, ref.batch(new, kv, 2, 1, 64, 16, torch.bfloat16, "cuda", pad=5))


def test_paged_attention_no_sequences(ops):
    s = ref.batch([2], [2], 2, 1, 64, 16, torch.bfloat16, "cuda")
    s["table"], s["lens"], s["cu"] = s["table"][:0], s["lens"][:0], s["cu"][:1]
    assert (attend(ops, s) == 0).all()
    s["q"] = s["q"][:0]
    assert attend(ops, s).shape == (0, 2, 64)


def test_paged_attention_more_tiles_than_the_card(ops):
    """so many rows that no tile's keys are split, and more than one round of them"""
    check(ops, ref.batch([300], [900], 160, 160, 64, 16, torch.bfloat16, "cuda"))
    check(ops, ref.batch([200, 5, 300], [200, 50, 700], 160, 160, 64, 16, torch.bfloat16, "cuda"))


@pytest.mark.parametrize("lens", [[3000, 2000, 100], [70000], [1] * 62 + [9000], [9000] + [1] * 200 + [300], [517] * 40])
@pytest.mark.parametrize("new", [1, 8, 33])
def test_paged_attention_many_splits(ops, lens, new):
    """more splits than the card takes at once, lengths far apart, more than 64 sequences"""
    kv = [max(n, new) for n in lens]
    check(ops, ref.batch([new] * len(kv), kv, 8, 2, 64, 16, torch.bfloat16, "cuda", pad=2))


@pytest.mark.parametrize("dtype,dim", [(torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 256), (torch.float32, 64)])
@pytest.mark.parametrize("count", [127, 128, 1100])
def test_paged_attention_hundreds_of_sequences(ops, dtype, dim, count):
    """single tokens, empty sequences, chunks and one long sequence among hundreds; rows behind the last"""
    new = [(1, 1, 0, 1, 3)[i % 5] for i in range(count)]
    kv = [n + (i * 37) % 70 for i, n in enumerate(new)]
    new[count // 2], kv[count // 2] = 60, 90
    kv[7] = 4000
    s = ref.batch(new, kv, 4, 2, dim, 16, dtype, "cuda", pad=40)
    check(ops, s)
    got = check(ops, s, window=33)
    assert (got[sum(new):] == 0).all()
    assert torch.equal(attend(ops, s, window=33), got)
    s = ref.batch([1] * count, [(i * 29) % 90 for i in range(count)], 4, 2, dim, 16, dtype, "cuda")
    check(ops, s)


def test_paged_attention_of_a_million_rows(ops):
    """2^20 tokens that see themselves only: the output is their value"""
    t, page = 1 << 20, 64
    pages = t // page + 2
    kc, vc = (torch.randn(pages, 1, page, 8, device="cuda").bfloat16() for _ in range(2))
    table = torch.randperm(pages, device="cuda").int()[None]
    q = torch.randn(t, 2, 8, device="cuda").bfloat16()
    got = ops.paged_attention(q, kc, vc, table, ints(0, t - 3), ints(t + 50), window=1)
    key = torch.arange(t - 3, device="cuda") + 53
    want = vc[table[0, key // page].long(), 0, key % page]
    assert torch.equal(got[:t - 3], want[:, None].expand(-1, 2, -1)) and (got[t - 3:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_paged_attention_empty_slots(ops, dtype):
    """a batch of fixed slots, most of them empty: prompts among them, as many tokens as slots"""
    new, kv = [0] * 400, [7] * 400
    for b, n, m in ((3, 1, 500), (70, 150, 150), (399, 130, 333), (200, 2, 2)):
        new[b], kv[b] = n, m
    check(ops, ref.batch(new, kv, 8, 2, 64, 16, dtype, "cuda", pad=1))
    check(ops, ref.batch([0, 0, 10, 0, 1, 0, 0, 0, 1, 0, 0, 0], [5, 0, 300, 9, 40, 1, 1, 1, 2, 0, 3, 3], 8, 1, 128, 16, dtype, "cuda"))


@pytest.mark.parametrize("new", [1, 100])
def test_paged_attention_many_small_weights(ops, new):
    """fp16: a hundred thousand keys whose weights are below fp16's values, beside one of weight 1.
    They are e^-17.4 = 2.8e-8 each (2^-25 and less is 0 in fp16), together 0.28 % of the sum."""
    n, page = 100000, 64
    s = ref.batch([new], [page], 4, 1, 64, page, torch.float16, "cuda")
    pages = n // page + 1
    s["kc"] = torch.zeros(pages, 1, page, 64, device="cuda", dtype=torch.float16)
    s["vc"] = torch.ones_like(s["kc"])
    s["kc"][0, 0, 0, 0], s["vc"][0, 0, 0] = 1.0, 0.0
    s["table"] = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    s["lens"] = ints(n)
    s["q"] = torch.zeros(new, 4, 64, device="cuda", dtype=torch.float16)
    s["q"][..., 0] = 17.4
    got = attend(ops, s, scale=1.0, causal=False).double()
    w = (n - 1) * torch.exp(-s["q"][0, 0, 0].double())
    want = w / (1 + w)
    # the weights are relative to 2^7 or more: off by at most 2^-12 each; the result by half a step
    assert (got / want - 1).abs().max() < 2.0 ** -12 + 2.0 ** -11 + 1e-5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [6, 200])
def test_paged_attention_hidden_values(ops, dtype, new):
    """an infinite or NaN value reaches the rows that see its key and no other"""
    s = ref.batch([new, 2], [new + 3, 12], 2, 1, 64, 4, dtype, "cuda")
    for key, x in ((new + 1, float("inf")), (new + 2, float("nan"))):
        s["vc"][s["table"][0, key // 4], :, key % 4] = x
    got = check(ops, s)
    assert got[:new - 2].isfinite().all() and not got[new - 2:new].isfinite().any() and got[new:].isfinite().all()
    s["kc"][s["table"][0, (new + 2) // 4], :, (new + 2) % 4] = float("nan")  # a key: only the last row's scores
    got = attend(ops, s)
    assert got[:new - 2].isfinite().all() and got[new - 1].isnan().all()
    got = attend(ops, s, window=2)
    assert got[:new - 2].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [2, 150])
def test_paged_attention_missing_pages(ops, dtype, new):
    s = ref.batch([new, 1], [new + 40, 60], 4, 2, 64, 16, dtype, "cuda")
    s["table"][0, 1], s["table"][0, 0], s["table"][1] = 100000, -5, -1
    got = check(ops, s)
    assert (got[new] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_attention_length_behind_the_table(ops, dtype):
    """a length of more pages than the table lists: the keys that are not there are hidden"""
    s = ref.batch([1, 70], [64, 70], 4, 2, 64, 16, dtype, "cuda")
    s["table"] = s["table"][:, :3].contiguous()
    check(ops, s)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("page", [1, 2, 3, 4, 12, 100])
def test_paged_attention_pages(ops, dim, page):
    """pages of any size in a batch that both forms share, rows behind the last sequence"""
    s = ref.batch([70, 1, 40, 3], [300, 200, 40, 133], 8, 2, dim, page, torch.bfloat16, "cuda", pad=30)
    got = check(ops, s)
    assert (got[114:] == 0).all()
    s = ref.batch([70], [300], 8, 2, dim, page, torch.float16, "cuda", pad=3)
    check(ops, s, window=90)


@pytest.mark.parametrize("new", [[1, 1], [80, 80], [1, 80]])
def test_paged_attention_shared_pages(ops, new):
    """sequences that share their pages: one table row for both"""
    s = ref.batch([80], [200], 8, 2, 128, 16, torch.bfloat16, "cuda")
    t = sum(new)
    s.update(table=s["table"].expand(2, -1), cu=ints(0, new[0], t), lens=ints(200, 190),
             q=torch.randn(t, 8, 128, device="cuda").bfloat16())
    got = check(ops, s)
    assert torch.equal(got, attend(ops, {**s, "table": s["table"].contiguous()}))


@pytest.mark.parametrize("new", [1, 120])
def test_paged_attention_wide_window(ops, new):
    s = ref.batch([new, 1], [130, 77], 4, 1, 64, 16, torch.bfloat16, "cuda")
    want = attend(ops, s)
    for window in (130, 2 ** 30 - 1, 2 ** 30, 2 ** 31, 2 ** 62):
        assert torch.equal(attend(ops, s, window=window), want), window


@pytest.mark.parametrize("new", [1, 120])
@pytest.mark.parametrize("window", [1, 2 ** 30 - 1, 2 ** 30, 2 ** 31 - 60, 2 ** 31 - 1, 2 ** 31, 2 ** 62])
def test_paged_attention_window_behind_the_table(ops, window, new):
    """lengths far behind the table: the window lies behind its keys, or reaches some or all of them"""
    s = ref.batch([new, 1], [130, 77], 4, 1, 64, 16, torch.float32, "cuda", stale=0.0)
    s["lens"] = ints(2 ** 31 - 1, 2 ** 31 - 40)
    for causal in (True, False):
        want = attend(ops, {n: t.cpu() for n, t in s.items()}, causal=causal, window=window)
        assert bool((want == 0).all()) == (window <= 2 ** 30)
        got = attend(ops, s, causal=causal, window=window)
        # (fp32 twice: scores of 64 products, at most 144 weights; all values below 8)
        assert (got.cpu() - want).abs().max() < 8 * (64 * 2 + 2 * 144 + 32) * 4 * ref.F32


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_attention_strides(ops, dtype):
    """token-major cache memory, a table row wider than its tensor, queries cut from a fused projection"""
    s = ref.batch([3, 150], [40, 170], 4, 2, 64, 16, dtype, "cuda", layout="tokens")
    assert not s["kc"].is_contiguous()
    wide = torch.full((2, 40), -1, dtype=torch.int32, device="cuda")
    wide[:, :s["table"].shape[1]] = s["table"]
    fused = torch.randn(153, 8, 64, device="cuda").to(dtype)
    fused[:, 2:6] = s["q"]
    want = check(ops, s)
    s.update(table=wide[:, :s["table"].shape[1]], q=fused[:, 2:6])
    assert torch.equal(attend(ops, s), want)
    odd = torch.zeros(153 * 4 * 64 + 1, device="cuda", dtype=dtype)[1:].view(153, 4, 64)  # (not 16-byte aligned)
    odd.copy_(s["q"])
    s["q"] = odd
    assert torch.equal(attend(ops, s), want)


def test_paged_attention_far_offsets(ops):
    """a cache of more than 2^31 elements; keys and values of one tensor"""
    page, hkv, dim = 64, 2, 128
    pages = (1 << 31) // (page * hkv * dim) + 200
    s = ref.batch([1, 150], [300, 333], 4, hkv, dim, page, torch.bfloat16, "cuda")
    big = torch.empty(pages, hkv, page, dim, device="cuda", dtype=torch.bfloat16)
    used = s["kc"].shape[0]
    big[pages - 2 * used:pages - used] = s["kc"]
    big[pages - used:] = s["vc"]
    small = attend(ops, s)
    table = torch.where(s["table"] >= 0, s["table"] + pages - 2 * used, -1).int()
    vc = big[used:]  # (the same page numbers)
    got = ops.paged_attention(s["q"], big[:pages - used], vc, table, s["cu"], s["lens"])
    assert torch.equal(got, small) and small.isfinite().all()


def test_paged_attention_is_repeatable(ops):
    for new, kv in (([1] * 9, [3000 + 77 * i for i in range(9)]), ([300, 40], [900, 2000])):
        s = ref.batch(new, kv, 8, 2, 128, 16, torch.bfloat16, "cuda")
        first = attend(ops, s)
        assert all(torch.equal(attend(ops, s), first) for _ in range(3))


def test_paged_attention_large_scores(ops):
    """scores of thousands: the maximum moves from block to block"""
    s = ref.batch([3, 160], [600, 160], 4, 2, 64, 16, torch.float32, "cuda")
    s["q"] *= 40
    check(ops, s)
    check(ops, s, scale=1e-3)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,kv", [(1, 70), (2, 9000), (9, 3000), (200, 200), (150, 3000)])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_paged_attention_scores_of_billions(ops, dtype, new, kv, dim):
    """Finite scores up to 2^31, either sign: a row is the mean of the values whose keys have its largest score.
    A score is one product of two values of 4 bits and less, so exact in fp32; two that differ do so by 2^19 at
    least (2^15 times the smallest step of the keys, 2^4), so the smaller one's weight is 0, and that of the largest
    is a power of two.  What is left: the sum of the values in fp32 and the rounding of the result."""
    s = ref.batch([new], [kv], 4, 2, dim, 16, dtype, "cuda", stale=0.0)
    gen = torch.Generator().manual_seed(new + kv)
    size = 2.0 ** torch.randint(8, 16, (2, kv), generator=gen)
    top = (torch.randint(8, 16, (2, kv), generator=gen) / 8 * size / 2).to(dtype).double()  # (4 bits each: many ties)
    at = s["table"][0].cpu()[torch.arange(kv) // 16].long()
    k = torch.zeros(kv, 2, dim, dtype=torch.float64)
    k[:, :, 3] = top.t()
    s["kc"][at.cuda(), :, (torch.arange(kv) % 16).cuda()] = k.to(dtype).cuda()
    v = s["vc"][at.cuda(), :, (torch.arange(kv) % 16).cuda()].double().cpu()  # [kv, 2, dim]
    s["q"].zero_()
    sign = torch.tensor([1.0, -1.0, 1.0, -1.0])
    s["q"][:, :, 3] = (sign * 2.0 ** 15).to(dtype).cuda()
    for causal in (True, False):
        got = attend(ops, s, scale=1.0, causal=causal).double().cpu()
        pos = torch.arange(kv - new, kv)[:, None]
        for h in range(4):
            score = (sign[h] * k[:, h // 2, 3]).expand(new, kv)
            if causal:
                score = score.masked_fill(torch.arange(kv) > pos, float("-inf"))
            w = (score == score.max(1, keepdim=True).values).double()
            want = w @ v[:, h // 2] / w.sum(1, keepdim=True)
            mag = w @ v[:, h // 2].abs() / w.sum(1, keepdim=True)
            ref.close(got[:, h], want, mag * (w.sum(1, keepdim=True) + 8) * ref.F32 + want.abs() * ref.half_step(dtype) + ref.smallest(dtype))


# ------------------------------------------------------- norm and rotation ----

SHAPES = [(1, 1, 8, 8), (4, 2, 64, 64), (3, 3, 40, 16), (8, 1, 128, 128), (5, 5, 72, 72), (2, 1, 256, 128), (32, 8, 128, 128),
          (3, 1, 192, 48), (100, 7, 96, 96), (6, 6, 80, 40)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk,dim,rot", SHAPES)
@pytest.mark.parametrize("inter", [False, True])
def test_qk_norm_rope(ops, dtype, hq, hk, dim, rot, inter):
    torch.manual_seed(dim + rot)
    q, k = (torch.randn(2, 37, hq, dim) * 3).to(dtype).cuda(), torch.randn(2, 37, hk, dim).to(dtype).cuda()
    qw, kw = torch.randn(dim).to(dtype).cuda(), torch.randn(dim).to(dtype).cuda()
    rope = ops.rope_table(50, rot).cuda()
    pos = torch.randint(0, 50, (2, 37)).cuda()
    pos[0, 3], pos[1, 0] = -1, 50
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    y = ops.qk_norm_rope(q, k, qw, kw, pos, rope, 1e-5, inter)
    gq, gk = torch.randn_like(y[0]), torch.randn_like(y[1])
    d = torch.autograd.grad(y, leaves, [gq, gk])
    for x, w, g, out, dx, dw in ((q, qw, gq, y[0], d[0], d[2]), (k, kw, gk, y[1], d[1], d[3])):
        ref.close(out, *ref.norm_rope(x, w, pos, rope, 1e-5, inter))
        want = ref.norm_rope_grad(x, w, g, pos, rope, 1e-5, inter)
        ref.close(dx, want[0], want[1])
        ref.close(dw, want[2], want[3])


def test_qk_norm_rope_empty_table(ops):
    q, k = (torch.randn(2, 3, n, 16, device="cuda", requires_grad=True) for n in (4, 2))
    w = torch.rand(16, device="cuda", requires_grad=True)
    for pos in (torch.tensor([[0, 1, 2], [5, -1, 0]], device="cuda"), torch.arange(3, device="cuda")):
        y = ops.qk_norm_rope(q, k, w, w, pos, ops.rope_table(0, 16).cuda())
        d = torch.autograd.grad(y, [q, k, w], [torch.ones_like(q), torch.ones_like(k)])
        assert [x.shape for x in d] == [q.shape, k.shape, w.shape] and not any(x.any() for x in (*y, *d))


@pytest.mark.parametrize("dtype", TYPES)
def test_qk_norm_rope_views(ops, dtype):
    """views of a fused projection, broadcast positions of either type, fp32 weights, one weight
    only, a broadcast gradient, rows that are only 8-byte aligned or not at all"""
    torch.manual_seed(1)
    rope, pos = ops.rope_table(20, 32).cuda(), torch.arange(5, 16, device="cuda")
    for offset in (0, 4, 1):
        store = torch.randn(3 * 11 * 9 * 64 + offset, device="cuda").to(dtype)[offset:]
        fused = store.view(3, 11, 9, 64)
        q, k = fused[:, :, :6].detach().requires_grad_(True), fused[:, :, 6:8].detach().requires_grad_(True)
        w = torch.randn(64, device="cuda", requires_grad=True)
        y = ops.qk_norm_rope(q, k, None, w, pos.int() if offset else pos, rope)
        full = pos.expand(3, 11)
        ref.close(y[0], *ref.norm_rope(q, None, full, rope, 1e-6, False))
        ref.close(y[1], *ref.norm_rope(k, w, full, rope, 1e-6, False))
        d = torch.autograd.grad(y[1].sum() + y[0][:, :, 1].float().sum(), [q, k, w])
        gq = torch.zeros(q.shape, device="cuda")
        gq[:, :, 1] = 1
        for x, ww, g, dx in ((q, None, gq, d[0]), (k, w, torch.ones(k.shape, device="cuda"), d[1])):
            want = ref.norm_rope_grad(x, ww, g, full, rope, 1e-6, False)
            ref.close(dx, want[0], want[1])
        ref.close(d[2], want[2], want[3])
        tokens = ops.qk_norm_rope(q[0], k[0], None, w, pos, rope)  # (three dimensions)
        assert torch.equal(tokens[0], y[0][0]) and torch.equal(tokens[1], y[1][0])


def test_qk_norm_rope_many_tokens(ops):
    """more tokens than the gradient's workgroups; the same sums every time; no tokens"""
    torch.manual_seed(2)
    q, k = torch.randn(4099, 6, 64, device="cuda"), torch.randn(4099, 2, 64, device="cuda")
    w = [torch.randn(64, device="cuda") for _ in range(2)]
    rope, pos = ops.rope_table(4099, 64).cuda(), torch.arange(4099, device="cuda")
    gq, gk = torch.randn_like(q), torch.randn_like(k)
    d = [ops.qk_norm_rope_backward(gq, gk, q, k, w[0], w[1], pos, rope) for _ in range(3)]
    assert all(torch.equal(a, b) for e in d[1:] for a, b in zip(d[0], e))
    for x, ww, g, dx, dw in ((q, w[0], gq, d[0][0], d[0][2]), (k, w[1], gk, d[0][1], d[0][3])):
        want = ref.norm_rope_grad(x, ww, g, pos, rope, 1e-6, False)
        ref.close(dx, want[0], want[1])
        ref.close(dw, want[2], want[3])
    e = ops.qk_norm_rope_backward(gq[:0], gk[:0], q[:0], k[:0], w[0], None, pos[:0], rope)
    assert e[0].shape == (0, 6, 64) and (e[2] == 0).all() and e[3].numel() == 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter,norm,rot", [(False, False, 0), (False, True, 16), (True, True, 24), (True, False, 8),
                                            (False, True, 24)])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_paged_append(ops, dtype, inter, norm, rot, layout):
    dim = 24
    s = ref.batch([3, 0, 1, 6, 2], [10, 4, 33, 5, 14], 6, 2, dim, 3, dtype, "cuda", pad=2, layout=layout)
    s["table"][4, 13 // 3] = 99
    rope = ops.rope_table(33, rot).cuda() if rot else None
    qw, kw = (torch.randn(dim, device="cuda"), torch.randn(dim, device="cuda")) if norm else (None, None)
    a = (s["table"], s["cu"], s["lens"], rope, norm, qw, kw, 1e-6, inter)
    want = ref.append(s["q"], s["k"], s["v"], s["kc"], s["vc"], *a)
    got = ops.paged_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], *a)
    for x, w in ((got, want[0]), (s["kc"], want[1]), (s["vc"], want[2])):
        ref.close(x, *w)
    again = s["kc"].clone()
    assert ops.paged_append(None, s["k"], s["v"], s["kc"], s["vc"], *a[:5], None, *a[6:]).numel() == 0
    assert torch.equal(s["kc"].nan_to_num(7.0), again.nan_to_num(7.0))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("dim,rot", [(24, 0), (24, 8), (64, 32), (128, 64), (128, 16), (72, 72)])
def test_infinite_values_stay_in_their_columns(ops, dtype, inter, dim, rot):
    """an infinite or NaN value reaches its own column and, within the rotated ones, the other of its pair"""
    tokens = 40
    gen = torch.Generator().manual_seed(dim + rot)
    x = torch.randn(tokens, 3, dim, generator=gen).to(dtype)
    for t in range(tokens):
        x[t, t % 3, t * 7 % dim] = (float("inf"), float("-inf"), float("nan"))[t // 3 % 3]
    x = x.cuda()
    table, cu, lens = ints(*range(4))[None], ints(0, tokens), ints(tokens)
    rope = ops.rope_table(tokens, rot).cuda() if rot else None
    kc, vc = (torch.zeros(4, 3, 16, dim, device="cuda", dtype=dtype) for _ in range(2))
    a = (table, cu, lens, rope, False, None, None, 1e-6, inter)
    if not rot:  # nothing is turned: a copy
        got = ops.paged_append(x, x, x, kc, vc, *a)
        flat = [c[:, h].reshape(64, dim)[:tokens] for c in (kc, vc) for h in range(3)]
        for y in (got, torch.stack(flat[:3], 1), torch.stack(flat[3:], 1)):
            ref.close(y, x, torch.zeros(x.shape))
        return
    want = ref.append(x, x, x, kc, vc, *a)
    got = ops.paged_append(x, x, x, kc, vc, *a)
    for y, w in ((got, want[0]), (kc, want[1]), (vc, want[2])):
        ref.close(y, *w)
    # with the norm an infinite value makes its row zero but for its own column and pair; the weights' gradient likewise
    g = torch.randn(tokens, 3, dim, generator=gen).to(dtype).cuda()
    g[5, 1, dim - 1], g[6, 0, 0] = float("inf"), float("-inf")
    x = x.nan_to_num(0.5, float("inf"), float("-inf"))
    w, pos = torch.rand(dim, generator=gen).cuda() + 0.5, torch.arange(tokens, device="cuda")
    for y in ops.qk_norm_rope(x, x, w, w, pos, rope, 1e-6, inter):
        ref.close(y, *ref.norm_rope(x, w, pos, rope, 1e-6, inter))
    clean = torch.randn(tokens, 3, dim, generator=gen).to(dtype).cuda()
    d = ops.qk_norm_rope_backward(g, g, clean, clean, w, w, pos, rope, 1e-6, inter)
    want = ref.norm_rope_grad(clean, w, g, pos, rope, 1e-6, inter)
    for dx, dw in ((d[0], d[2]), (d[1], d[3])):
        ref.close(dx, want[0], want[1])
        ref.close(dw, want[2], want[3])


@pytest.mark.parametrize("dtype", TYPES)
def test_paged_append_many_sequences(ops, dtype):
    new = [(i % 4) for i in range(300)]
    kv = [n + (i * 13) % 70 for i, n in enumerate(new)]
    s = ref.batch(new, kv, 8, 4, 128, 16, dtype, "cuda", pad=3)
    rope = ops.rope_table(100, 128).cuda()
    want = ref.append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], rope)
    got = ops.paged_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], rope)
    for x, w in ((got, want[0]), (s["kc"], want[1]), (s["vc"], want[2])):
        ref.close(x, *w)


def test_append_far_offsets(ops):
    page, hkv, dim = 64, 2, 128
    pages = (1 << 31) // (page * hkv * dim) + 8
    kc = torch.zeros(pages, hkv, page, dim, device="cuda", dtype=torch.bfloat16)
    k, v = (torch.randn(3, hkv, dim, device="cuda").bfloat16() for _ in range(2))
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda")
    cu, lens = torch.tensor([0, 3], dtype=torch.int32, device="cuda"), torch.tensor([66], dtype=torch.int32, device="cuda")
    vc = torch.zeros_like(kc)
    ops.paged_append(None, k, v, kc, vc, table, cu, lens)
    for c, x in ((kc, k), (vc, v)):
        assert torch.equal(c[pages - 1, :, 63], x[0]) and torch.equal(c[pages - 2, :, 0], x[1])
        assert torch.equal(c[pages - 2, :, 1], x[2]) and int((c != 0).any(-1).sum()) == 3 * hkv


# -------------------------------------------------------------- together ----

class Layer(torch.nn.Module):
    """A decoder layer's attention over a cache that it owns: fused rows [tokens, hq + 2 hkv, dim] in"""

    def __init__(self, hq: int, hkv: int, dim: int, page: int, table: torch.Tensor, pages: int, dtype: torch.dtype):
        super().__init__()
        self.hq, self.hkv = hq, hkv
        self.register_buffer("kc", torch.full((pages, hkv, page, dim), float("nan"), dtype=dtype))
        self.register_buffer("vc", torch.full((pages, hkv, page, dim), float("nan"), dtype=dtype))
        self.register_buffer("table", table)
        self.register_buffer("rope", torch.ops.nnsx.rope_table(4096, dim))
        self.register_buffer("qw", torch.linspace(0.5, 1.5, dim).to(dtype))
        self.register_buffer("kw", torch.linspace(1.5, 0.5, dim).to(dtype))

    def forward(self, x: torch.Tensor, cu: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
        q, k, v = x[:, :self.hq], x[:, self.hq:self.hq + self.hkv], x[:, self.hq + self.hkv:]
        q = torch.ops.nnsx.paged_append(q, k, v, self.kc, self.vc, self.table, cu, lens, self.rope, True, self.qw, self.kw)
        return torch.ops.nnsx.paged_attention(q, self.kc, self.vc, self.table, cu, lens)


def layer(dtype, sequences=2, hq=4, hkv=2, dim=64, page=16, width=30):
    table = torch.randperm(sequences * width).int().view(sequences, width)
    return Layer(hq, hkv, dim, page, table, sequences * width, dtype).cuda()


def ints(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def whole(m, xs):
    """the layer's definition over whole sequences, 64 bits after the append's rounding"""
    out = []
    for x in xs:
        pos = torch.arange(x.shape[0])
        q, _ = ref.norm_rope(x[:, :m.hq], m.qw, pos, m.rope, 1e-6, False)
        k, _ = ref.norm_rope(x[:, m.hq:m.hq + m.hkv], m.kw, pos, m.rope, 1e-6, False)
        q, k, v = (t.to(x.dtype).double() for t in (q, k, x[:, m.hq + m.hkv:].cpu()))
        rows = []
        for h in range(m.hq):
            g = h // (m.hq // m.hkv)
            s = q[:, h] @ k[:, g].t() / q.shape[-1] ** 0.5
            s = s.masked_fill(pos[None] > pos[:, None], float("-inf"))
            rows.append(torch.softmax(s, -1) @ v[:, g])
        out.append(torch.stack(rows, 1))
    return out


@pytest.mark.parametrize("dtype,tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2)])
def test_prompt_chunks_and_tokens_agree(ops, dtype, tol):
    """a prompt at once, in chunks and token by token fill the same cache and give the whole form's rows.
    (bf16: q and k rounded to 2^-8 twice over, scores of about 8 in magnitude, so weights off by about 3 %.)"""
    torch.manual_seed(5)
    xs = [torch.randn(n, 8, 64, device="cuda").to(dtype) for n in (310, 47)]
    outs = []
    for plan in ([(310, 47)], [(200, 40), (100, 0), (10, 7)], [(300, 30)] + [(1, 1)] * 9 + [(1, 8)]):
        m, at, got = layer(dtype), [0, 0], [[], []]
        torch.manual_seed(7)
        for step in plan:
            x = torch.cat([xs[b][at[b]:at[b] + n] for b, n in enumerate(step)])
            at = [a + n for a, n in zip(at, step)]
            y = m(x, ints(0, step[0], sum(step)), ints(*at))
            got[0].append(y[:step[0]])
            got[1].append(y[step[0]:])
        outs.append([torch.cat(g) for g in got])
    want = whole(m, xs)
    for o in outs:
        for a, b in zip(o, want):
            assert (a.double().cpu() - b).abs().max() < tol * max(1.0, b.abs().max().item())


def test_captured_graph_follows_the_lengths(ops):
    """one captured step replayed while the sequences grow, eager work between the replays"""
    torch.manual_seed(6)
    xs = torch.randn(40, 2, 8, 64, device="cuda").bfloat16()
    torch.manual_seed(8)
    a = layer(torch.bfloat16)
    torch.manual_seed(8)
    b = layer(torch.bfloat16)
    cu, lens, x = ints(0, 1, 2), ints(1, 1), xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a(x, cu, lens)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = a(x, cu, lens)
    for i in range(40):
        x.copy_(xs[i])
        lens.fill_(i + 1)
        graph.replay()
        want = b(xs[i], cu, ints(i + 1, i + 1))
        torch.cuda.synchronize()
        assert torch.equal(y, want), i
    assert torch.equal(a.kc.nan_to_num(9.0), b.kc.nan_to_num(9.0))


def test_two_graphs_and_an_eager_stream(ops):
    """calls of different shapes captured twice, replayed on two streams at once with eager calls beside them"""
    cases = [ref.batch([1] * 4, [900, 20, 333, 1], 8, 2, 128, 16, torch.bfloat16, "cuda"),
             ref.batch([1] * 3, [4000, 77, 1200], 8, 2, 128, 16, torch.bfloat16, "cuda", seed=4)]
    want = [attend(ops, s) for s in cases]
    graphs, outs = [], []
    for s in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(attend(ops, s))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[2]):
            eager = [attend(ops, s) for s in cases]
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert torch.equal(o, w) and torch.equal(e, w)
            o.zero_()


def test_captured_batches_of_any_kind(ops):
    """one graph for a number of tokens: single tokens, chunks and prompts among them from replay to replay"""
    kinds = [([120, 1, 1, 6], [400, 900, 33, 6]), ([1, 1, 1, 125], [100, 1, 500, 125]), ([32, 32, 32, 32], [900, 32, 70, 500]),
             ([0, 128, 0, 0], [5, 777, 0, 0]), ([1, 1, 1, 1], [900, 20, 300, 5]), ([0, 0, 0, 0], [0, 0, 0, 0])]
    s = ref.batch([32] * 4, [900] * 4, 8, 2, 128, 16, torch.bfloat16, "cuda")
    graph = torch.cuda.CUDAGraph()
    attend(ops, s)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = attend(ops, s)
    for new, kv in kinds + kinds[::-1]:
        s["cu"].copy_(ints(0, *torch.tensor(new).cumsum(0).tolist()))
        s["lens"].copy_(ints(*kv))
        graph.replay()
        want = attend(ops, {**s, "cu": s["cu"].clone(), "lens": s["lens"].clone()})
        torch.cuda.synchronize()
        assert torch.equal(out, want), new
        check(ops, s)
        out.fill_(7.0)


def test_captured_batch_of_many_sequences(ops):
    """as above with more sequences than a wave has lanes: slots that fill up, one long one among them"""
    count = 100
    s = ref.batch([2] * count, [40] * count, 8, 2, 64, 16, torch.bfloat16, "cuda")
    pool = torch.randn(400, 2, 16, 64, device="cuda").bfloat16()
    s.update(kc=pool, vc=torch.randn_like(pool), table=torch.randint(0, 400, (count, 200), device="cuda", dtype=torch.int32))
    graph = torch.cuda.CUDAGraph()
    attend(ops, s)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = attend(ops, s)
    for i in range(4):
        new = [(1, 0, 1, 2)[(b + i) % 4] for b in range(count)]
        new[i * 30] = 90
        kv = [n + (b * 17 + i) % 60 for b, n in enumerate(new)]
        kv[5 + i] += 3000
        s["cu"].copy_(ints(0, *torch.tensor(new).cumsum(0).tolist()))
        s["lens"].copy_(ints(*kv))
        graph.replay()
        want = attend(ops, {**s, "cu": s["cu"].clone(), "lens": s["lens"].clone()})
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        check(ops, s)
        out.fill_(7.0)


def test_captured_gradient(ops):
    """forward and backward of the norm in one graph, replayed over new inputs"""
    torch.manual_seed(9)
    q, k = torch.randn(70, 4, 64, device="cuda"), torch.randn(70, 2, 64, device="cuda")
    w = [torch.randn(64, device="cuda", requires_grad=True) for _ in range(2)]
    rope, pos = ops.rope_table(70, 64).cuda(), torch.arange(70, device="cuda")
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        a, b = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
        y = ops.qk_norm_rope(a, b, w[0], w[1], pos, rope)
        return list(y) + list(torch.autograd.grad(y, [a, b, w[0], w[1]], [gq, gk]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step()
    for i in range(4):
        q.normal_()
        gk.normal_()
        g.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, want)), i


def test_other_stream_and_inference_mode(ops):
    s = ref.batch([1, 40], [700, 50], 4, 2, 128, 16, torch.float16, "cuda")
    want = attend(ops, s)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st), torch.inference_mode():
        got = attend(ops, s)
    st.synchronize()
    assert torch.equal(got, want)


def test_refusals_across_devices(ops):
    s = ref.batch([1], [5], 2, 1, 64, 16, torch.bfloat16, "cuda")
    for name in ("kc", "vc", "table", "cu", "lens"):
        with pytest.raises(RuntimeError, match=" on "):
            attend(ops, {**s, name: s[name].cpu()})
    with pytest.raises(RuntimeError, match=" on "):
        ops.qk_norm_rope(s["q"], s["k"], None, None, torch.zeros(1, dtype=torch.int32), ops.rope_table(4, 64).cuda())
    with pytest.raises(RuntimeError, match=" on "):
        ops.qk_norm_rope(s["q"], s["k"], None, None, torch.zeros(1, dtype=torch.int32, device="cuda"), ops.rope_table(4, 64))


# ----------------------------------------------------------- in pipelines ----

class TokenModel(torch.nn.Module):
    """[1, hq + 2 hkv, dim] rows and the step's number in, the attention's row out"""

    def __init__(self, layer: Layer):
        super().__init__()
        self.layer = layer
        self.register_buffer("cu", torch.tensor([0, 1], dtype=torch.int32))

    def forward(self, x: torch.Tensor, n: torch.Tensor) -> torch.Tensor:
        return self.layer(x.view(1, 8, 64), self.cu, n.view(1)).reshape(1, 256)


@pytest.mark.parametrize("custom", ["hipgraph:true", "hipgraph:false"])
def test_token_model_in_a_pipeline(nns, tmp_path, custom):
    """tensor_filter runs the cache and the attention step by step, captured and eager"""
    import numpy as np

    torch.manual_seed(11)
    m = TokenModel(layer(torch.float32, sequences=1).cpu())
    xs = torch.randn(12, 8, 64)
    want = whole(m.layer, [xs])[0]
    path = str(tmp_path / "token.pt")
    torch.jit.script(m).save(path)
    caps = "other/tensors,format=static,num_tensors=2,dimensions=64:8:1.1,types=float32.int32,framerate=0/1"
    p = nns.parse_launch(f"appsrc name=src caps={caps} ! tensor_filter framework=pytorch model={path} "
                         f"accelerator=true:gpu device=0 custom={custom} ! tensor_sink name=s")
    got = []
    p.get_by_name("s").connect("new-data", lambda b: got.append(b.memory(0).numpy("float32").copy()))
    p.set_state("playing")
    for i in range(12):
        p.get_by_name("src").push_buffer([xs[i].numpy(), np.array([i + 1], dtype=np.int32)], pts=i)
    p.get_by_name("src").end_of_stream()
    p.wait(timeout=60)
    p.stop()
    assert len(got) == 12
    for i, g in enumerate(got):
        assert np.abs(g.reshape(4, 64) - want[i].numpy()).max() < 2e-5 * max(1.0, want[i].abs().max().item()), i


def test_trainer_on_gpu(nns, tmp_path):
    from test_attention import trained_weights

    trained_weights(nns, tmp_path, "device=0")
