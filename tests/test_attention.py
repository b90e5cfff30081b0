"""torch.ops.nnsx.qk_norm_rope / paged_append / paged_attention on the CPU: the
plain implementations that the kernels are compared with, and every refusal."""
import pytest
import torch

import attn_oracle as ref

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops(nns):
    return torch.ops.nnsx


def test_rope_table(ops):
    t = ops.rope_table(300000, 16, 10000.0)
    assert t.dtype == torch.float32 and t.shape == (300000, 16)
    ref.close(t, ref.table64(300000, 16), torch.full((300000, 16), 2.0 ** -24) + 1e-9)
    assert ops.rope_table(0, 8).shape == (0, 8)
    for bad in [(-1, 8, 1e4), (4, 7, 1e4), (4, 0, 1e4), (4, 8, 0.0), (4, 8, float("nan"))]:
        with pytest.raises(RuntimeError, match="rope_table"):
            ops.rope_table(*bad)


# heads of q and k, head dim, rotated columns
SHAPES = [(1, 1, 8, 8), (4, 2, 64, 64), (3, 3, 40, 16), (8, 1, 128, 128), (5, 5, 72, 72), (2, 1, 256, 128)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hk,dim,rot", SHAPES)
@pytest.mark.parametrize("inter", [False, True])
def test_qk_norm_rope(ops, dtype, hq, hk, dim, rot, inter):
    torch.manual_seed(dim + rot)
    q, k = (torch.randn(2, 7, hq, dim) * 3).to(dtype), torch.randn(2, 7, hk, dim).to(dtype)
    qw, kw = torch.randn(dim).to(dtype), torch.randn(dim).to(dtype)
    rope = ops.rope_table(50, rot)
    pos = torch.randint(0, 50, (2, 7))
    pos[0, 3], pos[1, 0] = -1, 50  # (not in the table: zero rows)
    y = ops.qk_norm_rope(q, k, qw, kw, pos, rope, 1e-5, inter)
    ref.close(y[0], *ref.norm_rope(q, qw, pos, rope, 1e-5, inter))
    ref.close(y[1], *ref.norm_rope(k, kw, pos, rope, 1e-5, inter))
    assert (y[0][0, 3] == 0).all() and (y[1][1, 0] == 0).all()


@pytest.mark.parametrize("inter", [False, True])
def test_qk_norm_rope_gradient(ops, inter):
    torch.manual_seed(3)
    q, k = torch.randn(5, 3, 24), torch.randn(5, 2, 24)
    qw, kw = torch.randn(24), torch.randn(24)
    rope, pos = ops.rope_table(9, 16), torch.tensor([0, 3, -1, 8, 9], dtype=torch.int32)
    leaves = [t.requires_grad_(True) for t in (q, k, qw, kw)]
    y = ops.qk_norm_rope(q, k, qw, kw, pos, rope, 1e-4, inter)
    gq, gk = torch.randn_like(y[0]), torch.randn_like(y[1])
    d = torch.autograd.grad(y, leaves, [gq, gk])
    for x, w, g, dx, dw in ((q, qw, gq, d[0], d[2]), (k, kw, gk, d[1], d[3])):
        want = ref.norm_rope_grad(x, w, g, pos, rope, 1e-4, inter)
        ref.close(dx, want[0], want[1])
        ref.close(dw, want[2], want[3])
    # and against differences of the 64-bit form: central, error h^2 / 6 of the third derivative plus rounding / h
    h = 1e-5
    for leaf, got in ((q, d[0]), (qw, d[2])):
        flat = leaf.detach().double()
        for i in [0, 7, 20, flat.numel() - 1]:
            val = []
            for s in (h, -h):
                t = flat.clone().view(-1)
                t[i] += s
                t = t.view(flat.shape)
                x, w = (t, qw) if leaf is q else (q, t)
                val.append((ref.norm_rope(x, w, pos, rope, 1e-4, inter)[0] * gq.double()).sum())
            want = (val[0] - val[1]) / (2 * h)
            assert abs(got.reshape(-1)[i].item() - want.item()) < 1e-4 * max(1.0, abs(want.item()))


def test_qk_norm_rope_gradient_without_weights_and_second_order(ops):
    q, k = torch.randn(4, 2, 8, requires_grad=True), torch.randn(4, 1, 8, requires_grad=True)
    rope, pos = ops.rope_table(4, 8), torch.arange(4)
    y = ops.qk_norm_rope(q, k, None, None, pos, rope)
    d = torch.autograd.grad(y[0].sum(), q, retain_graph=True)[0]  # (k's output unused)
    want = ref.norm_rope_grad(q, None, torch.ones_like(q), pos, rope, 1e-6, False)
    ref.close(d, want[0], want[1])
    with pytest.raises(RuntimeError, match="no gradient"):
        torch.autograd.grad(y[0].sum(), q, create_graph=True)


def test_qk_norm_rope_empty_table(ops):
    """no position is in a table of none: zero rows, zero gradients, whatever the positions' shape"""
    for shape, positions in (((2, 3), torch.tensor([[0, 1, 2], [5, -1, 0]])), ((2, 3), torch.arange(3)), ((3,), torch.arange(3))):
        q, k = (torch.randn(*shape, n, 16, requires_grad=True) for n in (4, 2))
        w = torch.rand(16, requires_grad=True)
        y = ops.qk_norm_rope(q, k, w, w, positions, ops.rope_table(0, 16))
        assert y[0].shape == q.shape and y[1].shape == k.shape and not y[0].any() and not y[1].any()
        d = torch.autograd.grad(y, [q, k, w], [torch.ones_like(q), torch.ones_like(k)])
        assert [x.shape for x in d] == [q.shape, k.shape, w.shape] and not any(x.any() for x in d)


BATCHES = [
    ([1], [1], 1, 1, 8, 4), ([1], [0], 2, 1, 8, 4), ([0], [5], 2, 1, 8, 4), ([5], [3], 2, 2, 16, 4),
    ([3, 0, 1, 6], [10, 4, 33, 6], 6, 2, 24, 3), ([2, 9], [70, 9], 4, 4, 32, 1), ([4, 1], [20, 64], 8, 1, 64, 16),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new,kv,hq,hkv,dim,page", BATCHES)
@pytest.mark.parametrize("causal,window", [(True, 0), (True, 3), (False, 0), (False, 2)])
def test_paged_attention(ops, dtype, new, kv, hq, hkv, dim, page, causal, window):
    s = ref.batch(new, kv, hq, hkv, dim, page, dtype, pad=2, seed=len(new) + dim)
    got = ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], causal=causal, window=window)
    ref.close(got, *ref.attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], None, causal, window))
    assert (got[sum(new):] == 0).all()


def test_paged_attention_hidden_values_and_missing_pages(ops):
    s = ref.batch([6, 2], [9, 12], 2, 1, 16, 4, torch.float32)
    for i in (7, 8):  # the last two tokens' values: earlier rows must not see them
        s["vc"][s["table"][0, i // 4], :, i % 4] = float("inf") if i == 7 else float("nan")
    s["table"][1, 1] = 1000  # (not a page of the cache)
    s["table"][1, 0] = -7
    got = ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"])
    ref.close(got, *ref.attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"]))
    assert got[:4].isfinite().all() and not got[4:6].isfinite().any() and got[6:].isfinite().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("inter,norm,rot", [(False, False, 0), (False, True, 16), (True, True, 24), (True, False, 8)])
def test_paged_append(ops, dtype, inter, norm, rot):
    dim = 24
    s = ref.batch([3, 0, 1, 6, 2], [10, 4, 33, 5, 14], 6, 2, dim, 3, dtype, pad=2)
    s["table"][4, 13 // 3] = 99  # (its last token has no page)
    rope = ops.rope_table(33, rot) if rot else None  # (position 32 is the last)
    qw, kw = (torch.randn(dim).to(dtype), torch.randn(dim)) if norm else (None, None)
    if norm:
        qw = qw.float()
    want = ref.append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], rope, norm, qw, kw, 1e-6, inter)
    got = ops.paged_append(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], rope, norm, qw, kw, 1e-6, inter)
    ref.close(got, *want[0])
    ref.close(s["kc"], *want[1])
    ref.close(s["vc"], *want[2])


def test_paged_append_without_queries(ops):
    s = ref.batch([2], [5], 2, 2, 8, 4, torch.float32)
    want = ref.append(None, s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"])
    got = ops.paged_append(None, s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"])
    assert got.shape == (0,)
    ref.close(s["kc"], *want[1])
    ref.close(s["vc"], *want[2])


def refused(match, f, *a, **k):
    with pytest.raises(RuntimeError, match=match):
        f(*a, **k)


def test_refusals_of_the_cache_and_the_batch(ops):
    def call(**over):
        s = {**ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32), **over}
        return ops.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], **{
            k: v for k, v in over.items() if k in ("scale", "window")})

    s = ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32)
    call()
    refused("q is", call, q=s["q"][0])
    refused("bfloat16, float16 or float32", call, q=s["q"].double())
    refused("k_cache is", call, kc=s["kc"].half())
    refused("v_cache is", call, vc=s["vc"].bfloat16())
    refused("both", call, vc=s["vc"][:, :, :3])
    refused("both", call, kc=s["kc"][0], vc=s["vc"][0])
    refused("does not fit", call, q=s["q"][:, :3])
    refused("does not fit", call, q=s["q"][:, :, :8].contiguous())
    refused("rows of the cache", call, kc=s["kc"].transpose(2, 3).contiguous().transpose(2, 3))
    wide = torch.zeros(s["kc"].shape[:3] + (17,))
    refused("rows of the cache", call, kc=wide[..., :16])
    refused("head dim", call, q=s["q"][..., :12], kc=s["kc"][..., :12], vc=s["vc"][..., :12])
    big = torch.zeros(2, 2, 4, 264)
    refused("head dim", call, q=torch.zeros(3, 4, 264), kc=big, vc=big)
    refused("page_table", call, table=s["table"].long())
    refused("page_table", call, table=s["table"][0])
    refused("page_table", call, table=torch.zeros(2, 6, dtype=torch.int32)[:, ::2])
    refused("kv_lens", call, lens=s["lens"][:1])
    refused("kv_lens", call, lens=s["lens"].long())
    refused("cu_seqlens", call, cu=s["cu"][:2])
    refused("starts with 0", call, cu=torch.tensor([1, 2, 3], dtype=torch.int32))
    refused("ascends", call, cu=torch.tensor([0, 2, 1], dtype=torch.int32))
    refused("ascends", call, cu=torch.tensor([0, 2, 4], dtype=torch.int32))
    refused("no heads", call, kc=s["kc"][:, :0], vc=s["vc"][:, :0])
    for bad in (0.0, -1.0, float("inf"), float("nan"), 1e-60):
        refused("scale", call, scale=bad)
    refused("window", call, window=-1)
    refused("no gradient", call, q=s["q"].requires_grad_(True))
    with torch.no_grad():
        call(q=s["q"])
        far = torch.empty_strided((2, 2, 4, 16), (2 ** 29 + 4, 64, 16, 1))  # (never touched)
        refused("apart", call, kc=far, vc=far)
        far = torch.empty_strided((2, 2, 4, 16), (32, 16, 2 ** 26 + 64, 1))
        refused("apart", call, kc=far, vc=far)
        refused("more than one call takes", call, q=s["q"][:1].expand(2 ** 23, 4, 16))
        empty = torch.empty(0, 2, 2 ** 31 + 4, 16)
        refused("more than one call takes", call, kc=empty, vc=empty, table=torch.empty(2, 0, dtype=torch.int32))
        refused("more than one call takes", call, table=torch.empty_strided((2, 2 ** 28 + 1), (1, 1), dtype=torch.int32))


def test_refusals_of_append(ops):
    s = ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32)
    rope, w = ops.rope_table(9, 16), torch.ones(16)

    def call(q=s["q"], k=s["k"], v=s["v"], kc=s["kc"], vc=s["vc"], **over):
        return ops.paged_append(q, k, v, kc, vc, s["table"], s["cu"], s["lens"], **over)

    call(rope=rope)
    refused("k and v", call, k=s["k"][0])
    refused("k and v", call, v=s["v"][:2])
    refused("v is", call, v=s["v"].half())
    refused("k_cache is", call, kc=s["kc"].half())
    refused("does not fit a cache", call, k=s["k"][:, :1], v=s["v"][:, :1])
    refused("does not fit k", call, q=s["q"][:2])
    refused("q is", call, q=s["q"].half())
    refused("float32 table", call, rope=rope.double())
    refused("rotated columns", call, rope=rope[:, :12].contiguous())
    refused("rotated columns", call, rope=ops.rope_table(9, 24))
    refused("weights without norm", call, k_weight=w)
    refused("q_weight without q", call, q=None, norm=True, q_weight=w)
    refused("k_weight is", call, norm=True, k_weight=torch.ones(8))
    refused("one type", ops.paged_append, s["q"].half(), s["k"].half(), s["v"].half(), s["kc"].half(), s["vc"].half(),
            s["table"], s["cu"], s["lens"], norm=True, q_weight=w, k_weight=w.half())
    refused("eps", call, norm=True, eps=-1.0)
    refused("lie on each other", call, kc=s["kc"][:1].expand(s["kc"].shape))
    refused("are one", call, vc=s["kc"])
    pool = torch.zeros(s["kc"].numel() * 2)
    part = pool[:s["kc"].numel()].view(s["kc"].shape)
    refused("are one", call, kc=part, vc=pool[8:8 + s["kc"].numel()].view(s["kc"].shape))
    refused("part of the cache", call, kc=part, vc=pool[s["kc"].numel():].view(s["kc"].shape), k=pool[:s["k"].numel()].view(s["k"].shape))
    call(kc=part, vc=pool[s["kc"].numel():].view(s["kc"].shape))
    refused("no gradient", call, k=s["k"].clone().requires_grad_(True))
    refused("no gradient", call, rope=rope.clone().requires_grad_(True))


def test_qk_norm_rope_part_of_the_gradient(ops):
    """one output used, inputs that ask for none, the graph used twice and given back"""
    torch.manual_seed(3)
    q, k, w = torch.randn(5, 4, 16), torch.randn(5, 2, 16), torch.rand(16) + 0.5
    pos, rope = torch.arange(5), ops.rope_table(5, 16)
    g = torch.randn(5, 2, 16)
    full = ops.qk_norm_rope_backward(torch.zeros_like(q), g, q, k, w, w, pos, rope)
    a = [x.clone().requires_grad_(True) for x in (q, k, w, w)]
    _, yk = ops.qk_norm_rope(*a, pos, rope)
    got = torch.autograd.grad(yk, a, g, retain_graph=True)
    assert all(torch.equal(x, y) for x, y in zip(got, full)) and (got[0] == 0).all()
    assert torch.equal(torch.autograd.grad(yk, a[1], g)[0], full[1])
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(yk, a[1], g)
    k2 = k.clone().requires_grad_(True)
    yq, yk = ops.qk_norm_rope(q, k2, None, w, pos, rope)
    assert yq.requires_grad and yk.requires_grad
    yk.backward(g)
    assert torch.equal(k2.grad, full[1]) and q.grad is None
    k2 = k.clone().requires_grad_(True)
    _, yk = ops.qk_norm_rope(q, k2 * 1.0, None, None, pos, rope)
    assert not ops.qk_norm_rope(q, k, w, w, pos, rope)[0].requires_grad
    with torch.no_grad():
        assert not ops.qk_norm_rope(q, k2, w, w, pos, rope)[1].requires_grad
    x = k.clone().requires_grad_(True) * 1.0
    _, yk = ops.qk_norm_rope(q, x, None, None, pos, rope)
    x.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        yk.sum().backward()


def test_append_to_a_cache_of_inference_mode(ops):
    """outside that mode it is refused before a row is written"""
    s = ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32, stale=0.0)
    with torch.inference_mode():
        kc, vc = s["kc"].clone(), s["vc"].clone()
    a = (s["k"], s["v"]), (s["table"], s["cu"], s["lens"])
    for k, v in ((kc, s["vc"]), (s["kc"], vc)):
        before = k.clone(), v.clone()
        refused("inference mode", ops.paged_append, None, *a[0], k, v, *a[1])
        assert torch.equal(k, before[0]) and torch.equal(v, before[1])
    with torch.inference_mode():
        ops.paged_append(None, *a[0], kc, vc, *a[1])
        assert not torch.equal(kc, s["kc"])


def test_forward_mode_is_refused(ops):
    """a tangent is not dropped unnoticed, under no_grad neither"""
    import torch.autograd.forward_ad as fw

    s = ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32)
    rope, pos, w, q, k = ops.rope_table(9, 16), torch.arange(3), torch.ones(16), s["q"], s["k"]
    with fw.dual_level(), torch.no_grad():
        def dual(x):
            return fw.make_dual(x, torch.ones_like(x))

        for a in ((dual(q), s["kc"], s["vc"]), (q, dual(s["kc"]), s["vc"]), (q, s["kc"], dual(s["vc"]))):
            refused("no forward-mode gradient", ops.paged_attention, *a, s["table"], s["cu"], s["lens"])
        for a in ((dual(q), k, s["v"], rope), (q, dual(k), s["v"], rope), (q, k, dual(s["v"]), rope), (q, k, s["v"], dual(rope))):
            refused("no forward-mode gradient", ops.paged_append, *a[:3], s["kc"], s["vc"], s["table"], s["cu"], s["lens"], a[3])
        for a in ((dual(q), k, w, rope), (q, k, dual(w), rope), (q, k, w, dual(rope))):
            refused("no forward-mode gradient", ops.qk_norm_rope, a[0], a[1], a[2], None, pos, a[3])
        refused("no forward-mode gradient", ops.qk_norm_rope_backward, dual(q), k, q, k, None, None, pos, rope)


def test_append_is_seen_by_gradients(ops):
    """a cache that an earlier operation keeps for its gradient is not changed unnoticed"""
    s = ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32)
    w = torch.ones(16, requires_grad=True)
    loss = (s["kc"] * w).sum()
    ops.paged_append(None, s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"])
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    with torch.inference_mode():
        s = ref.batch([2, 1], [5, 9], 4, 2, 16, 4, torch.float32)
        ops.paged_append(None, s["k"], s["v"], s["kc"], s["vc"], s["table"], s["cu"], s["lens"])


def test_refusals_of_norm_rope(ops):
    q, k, pos, rope = torch.randn(3, 4, 16), torch.randn(3, 2, 16), torch.arange(3), ops.rope_table(4, 16)

    def call(q=q, k=k, qw=None, kw=None, pos=pos, rope=rope, eps=1e-6):
        return ops.qk_norm_rope(q, k, qw, kw, pos, rope, eps)

    call()
    refused("bfloat16, float16 or float32", call, q=q.double(), k=k.double())
    refused("k is", call, k=k.half())
    refused("q and k are both", call, q=q[0], k=k[0])
    refused("differ", call, k=k[:2])
    refused("differ", call, k=k[:, :, :8])
    refused("differ", call, k=k[:, :0])
    refused("head dim", call, q=q[..., :12], k=k[..., :12])
    refused("rotated", call, rope=ops.rope_table(4, 24))
    refused("float32 table", call, rope=rope.half())
    refused("positions", call, pos=pos.float())
    refused("positions", call, pos=pos[:2])
    refused("positions", call, pos=pos[None])
    refused("q_weight", call, qw=torch.ones(8))
    refused("k_weight", call, kw=torch.ones(16).half())
    refused("no gradient", call, rope=rope.clone().requires_grad_(True))
    refused("eps", call, eps=float("nan"))
    refused("more tokens", call, q=q[:1].expand(2 ** 23, 4, 16), k=k[:1].expand(2 ** 23, 2, 16), pos=pos[:1].expand(2 ** 23))


def test_script(ops):
    """a TorchScript module calls them, as tensor_filter's models do"""

    class Layer(torch.nn.Module):
        def __init__(self):
            super().__init__()
            s = ref.batch([1], [3], 2, 1, 8, 4, torch.float32)
            self.register_buffer("kc", s["kc"])
            self.register_buffer("vc", s["vc"])
            self.register_buffer("table", s["table"])
            self.register_buffer("cu", s["cu"])
            self.register_buffer("rope", torch.ops.nnsx.rope_table(16, 8))

        def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lens: torch.Tensor) -> torch.Tensor:
            q = torch.ops.nnsx.paged_append(q, k, v, self.kc, self.vc, self.table, self.cu, lens, self.rope, True)
            return torch.ops.nnsx.paged_attention(q, self.kc, self.vc, self.table, self.cu, lens)

    m = Layer()
    q, k, v, lens = torch.randn(1, 2, 8), torch.randn(1, 1, 8), torch.randn(1, 1, 8), torch.tensor([3], dtype=torch.int32)
    want = m(q, k, v, lens)
    assert torch.equal(torch.jit.script(m)(q, k, v, lens), want) and want.isfinite().all()


class Scorer(torch.nn.Module):
    """rows [n, 5 * 3 * 8] -> scores [n, 8] through the per-head norm and rotation, with trained norm weights"""

    def __init__(self):
        super().__init__()
        self.qw = torch.nn.Parameter(torch.linspace(0.5, 1.5, 8))
        self.kw = torch.nn.Parameter(torch.linspace(1.5, 0.5, 8))
        self.register_buffer("rope", torch.ops.nnsx.rope_table(5, 8))
        self.register_buffer("pos", torch.arange(5))

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        x = x.view(-1, 5, 3, 8)
        q, k = torch.ops.nnsx.qk_norm_rope(x[:, :, :2], x[:, :, 2:], self.qw, self.kw, self.pos, self.rope)
        return q.sum([1, 2]) + 0.5 * k.sum([1, 2])


def trained_weights(nns, tmp_path, device):
    """one step of tensor_trainer's plain gradient descent moves the weights by the gradient's definition"""
    import numpy as np

    torch.manual_seed(4)
    m = Scorer()
    torch.jit.script(m).save(str(tmp_path / "scorer.pt"))
    (tmp_path / "scorer.ini").write_text(f"model = {tmp_path}/scorer.pt\nloss = cross_entropy\noptimizer = sgd\n"
                                         "learning_rate = 0.5\nbatch_size = 6\n")
    xs, labels = torch.randn(6, 120), torch.arange(6)
    caps = "other/tensors,format=static,num_tensors=2,dimensions=120:1.1:1,types=float32.int32,framerate=0/1"
    p = nns.parse_launch(
        f"appsrc name=src caps={caps} ! tensor_trainer name=tr framework=pytorch model-config={tmp_path}/scorer.ini "
        f"model-save-path={tmp_path}/out.pt num-inputs=1 num-labels=1 num-training-samples=6 num-validation-samples=0 "
        f"epochs=1 {device} ! tensor_sink name=s")
    p.set_state("playing")
    for i in range(6):
        p.get_by_name("src").push_buffer([xs[i].numpy(), np.array([i], np.int32)], pts=i)
    p.get_by_name("src").end_of_stream()
    msg = p.wait(60)
    p.stop()
    assert msg and msg[0] == "eos", p.messages()
    after = torch.jit.load(str(tmp_path / "out.pt"), map_location="cpu")
    x, rope = xs.double().view(6, 5, 3, 8), m.rope.double()
    q, k, pos = x[:, :, :2].float(), x[:, :, 2:].float(), torch.arange(5).expand(6, 5)
    yq, yk = (ref.norm_rope(a, w, pos, rope, 1e-6, False)[0] for a, w in ((q, m.qw), (k, m.kw)))
    prob = torch.softmax(yq.sum([1, 2]) + 0.5 * yk.sum([1, 2]), -1)
    g = (prob - torch.nn.functional.one_hot(labels, 8)) / 6
    for w, x0, f, got in ((m.qw, q, 1.0, after.qw), (m.kw, k, 0.5, after.kw)):
        dw = ref.norm_rope_grad(x0, w, (g * f)[:, None, None].expand(x0.shape), pos, rope, 1e-6, False)[2]
        # every term carries fewer than 100 roundings of 2^-24 on sums of 60 terms of about 1
        assert dw.abs().max() > 0.01 and (got.double() - (w.double() - 0.5 * dw)).abs().max() < 1e-4


def test_trainer(nns, tmp_path):
    trained_weights(nns, tmp_path, "")
