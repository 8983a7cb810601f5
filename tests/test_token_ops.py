"""Embedding rows by token (ops.token_embed) and attention over chosen key blocks (ops.block_keys, block_select,
block_attention, sparse_attention), each against the definition in 64 bits.

Tolerances count roundings. bf16 rounds by at most 2^-8 of a value (half a step), fp32 by 2^-24. An attention weight p is
exact to 2^-12 (fp32 scores of at most 64 products, whose size the inputs here keep below 2^6, the fast exponential) and is
rounded to bf16 where the matrix cores take it as an operand; so is ds. With sums of absolute terms in the reference:
  out  2^-8 |out| + (2^-8 + 2^-12) sum p |v|
  dv   2^-8 |dv|  + (2^-8 + 2^-12) sum p |do|
  dq   2^-8 |dq|  + (2^-8 + 2^-11) sum |ds| |k| + scale * sum p |k| * E    (dk: the same over queries, with q)
  E    the error of do . v - delta: 2^-15 |do| . |out| (delta's operand is a pair of bf16 numbers) + 2^-17 max |do| . |v|
       + (2^-8 + 2^-12) sum p |do . v - delta|: out = sum P v / sum P with P = p (1 + e), |e| <= 2^-8, is off by
       sum p e (v - out) / sum P, and delta = do . out by that times do
The table's gradient is an fp32 sum of n terms: n 2^-24 sum |terms|, at least two roundings."""
import ctypes

import pytest
import torch

from tests.parity import rel_err  # noqa: F401  (one place for the tests' path set-up)

gpu = pytest.mark.gpu
H = 2.0 ** -8
BLOCK = 64


def ops():
    from dm_hip import ops as o
    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(torch.bfloat16)


@pytest.fixture(autouse=True)
def _pool_by_shape():
    yield
    from dm_hip import ops as o
    o.BLOCK_POOL = 0


def rows_together(n):
    """how many rows a workgroup takes: by the shape (0), one query (1), or a pool on the matrix cores"""
    ops().BLOCK_POOL = n


# -------------------------------------------------------------------------------------------------- references
def lengths(k_len, B, L):
    return torch.full((B,), L, device="cuda") if k_len is None else k_len.clamp(0, L)


def ref_keys(k, k_len):
    B, L, Hk, D = k.shape
    n = -(-L // BLOCK)
    out = torch.zeros(B, Hk, n, D, dtype=torch.float64, device="cuda")
    for b, have in enumerate(lengths(k_len, B, L).tolist()):
        for j in range(-(-have // BLOCK)):
            out[b, :, j] = k[b, j * BLOCK:min(have, (j + 1) * BLOCK)].double().mean(0)
    return out


def ref_select(q, keys, top, k_len, L):
    """the best blocks by (score, -block), one query after another as sorted lists"""
    B, Lq, Hq, D = q.shape
    score = torch.einsum("bihd,bhjd->bhij", q.double(), keys.double().repeat_interleave(Hq // keys.shape[1], 1))
    score = torch.nan_to_num(score, nan=-float("inf"), posinf=float("inf"), neginf=-float("inf")).cpu()
    out = torch.full((B, Hq, Lq, top), -1, dtype=torch.int32)
    for b, have in enumerate(lengths(k_len, B, L).tolist()):
        n = -(-have // BLOCK)
        for h in range(Hq):
            for i in range(Lq):
                row = score[b, h, i, :n].tolist()
                best = sorted(sorted(range(n), key=lambda j: (-row[j], j))[:top])
                out[b, h, i, :len(best)] = torch.tensor(best, dtype=torch.int32)
    return out.cuda()


def ref_attention(q, k, v, blocks, scale, k_len, dout):
    """(out, dq, dk, dv) in 64 bits and the bound of each, as in the module's text"""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    G, n = Hq // Hkv, -(-Lk // BLOCK)
    t = lambda x: x.double().transpose(1, 2)                                     # noqa: E731
    have = lengths(k_len, B, Lk)
    pos = torch.arange(Lk, device="cuda")
    ok = (pos < have[:, None])[:, None, :, None]
    qs, do = t(q), t(dout)
    ks, vs = (torch.where(ok, t(x), 0.0).repeat_interleave(G, 1) for x in (k, v))
    seen = torch.zeros(B, Hq, Lq, n, dtype=torch.bool, device="cuda")
    for c in range(blocks.shape[3]):
        j = blocks[..., c].long()
        good = (j >= 0) & (j < n)
        seen |= good[..., None] & (torch.arange(n, device="cuda") == j[..., None])
    seen = seen.repeat_interleave(BLOCK, 3)[..., :Lk] & ok.transpose(2, 3)
    s = torch.where(seen, torch.matmul(qs, ks.transpose(2, 3)) * scale, -float("inf"))
    p = torch.where(seen.any(-1, keepdim=True), torch.softmax(s, -1), 0.0)
    out = torch.matmul(p, vs)
    dp = torch.matmul(do, vs.transpose(2, 3))
    ds = p * (dp - (do * out).sum(-1, keepdim=True)) * scale
    back = lambda x: x.transpose(1, 2)                                           # noqa: E731
    keys = lambda x: x.view(B, Hkv, G, Lk, D).sum(2).transpose(1, 2)             # noqa: E731
    T = lambda x: x.transpose(2, 3)                                              # noqa: E731
    dq, dk, dv = torch.matmul(ds, ks), torch.matmul(T(ds), qs), torch.matmul(T(p), do)
    E = 2.0 ** -15 * (do.abs() * out.abs()).sum(-1, keepdim=True) + 2.0 ** -17 * torch.where(seen, torch.matmul(do.abs(), T(vs.abs())), 0.0).amax(-1, keepdim=True)
    E = E + (H + 2.0 ** -12) * (p * (dp - (do * out).sum(-1, keepdim=True))).abs().sum(-1, keepdim=True)
    w, e = ds.abs() * (H + 2.0 ** -11), abs(scale) * p * E
    tiny = 1e-30
    return ((back(out), back(H * out.abs() + (H + 2.0 ** -12) * torch.matmul(p, vs.abs()) + tiny)),
            (back(dq), back(H * dq.abs() + torch.matmul(w + e, ks.abs()) + tiny)),
            (keys(dk), H * keys(dk).abs() + keys(torch.matmul(T(w + e), qs.abs())) + tiny),
            (keys(dv), H * keys(dv).abs() + (H + 2.0 ** -12) * keys(torch.matmul(T(p), do.abs())) + tiny))


def within(name, got, want, bound):
    over = (got.detach().double() - want).abs() / bound
    assert bool(torch.isfinite(got.double()).all()), f"{name}: not finite"
    assert float(over.max()) <= 1.0, f"{name}: {float(over.max()):.3g} of the bound at {int(over.argmax())}"


def some_blocks(g, B, Hq, Lq, n, top):
    """any list a caller may hand over: repeats, -1 and numbers that are no block among them"""
    b = torch.randint(-1, n + 1, (B, Hq, Lq, top), generator=g, device="cuda", dtype=torch.int32)
    b[torch.rand(B, Hq, Lq, generator=g, device="cuda") < 0.1] = -1   # queries without a block
    return b


# -------------------------------------------------------------------------------------------------- choice of blocks
@gpu
@pytest.mark.parametrize("pool", [0, 1, 512])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,top,ragged", [
    (1, 1, 1, 1, 1, 8, 1, False),
    (2, 5, 63, 2, 1, 16, 3, False),
    (2, 7, 64, 4, 4, 8, 2, False),
    (3, 70, 65, 2, 2, 32, 1, True),
    (3, 65, 1000, 6, 3, 64, 5, True),
    (1, 130, 4200, 2, 1, 64, 16, False),     # more than 64 blocks
    (2, 33, 9000, 2, 2, 8, 64, True),
    (1, 3, 300, 40, 40, 16, 9, False),       # more heads than one workgroup's 64 vectors hold; top above the block count
    (1, 2, 70000, 1, 1, 8, 20, False),       # more blocks than are scored at a time, few queries
    (1, 20, 70000, 1, 1, 8, 10, False),      # ... and more
    (2, 9, 5000, 4, 2, 32, 30, True),
    (1, 17, 5000, 2, 2, 16, 60, False),
])
def test_block_choice(B, Lq, Lk, Hq, Hkv, D, top, ragged, pool):
    rows_together(pool)
    g = gen(1)
    q, k = randn(g, B, Lq, Hq, D), randn(g, B, Lk, Hkv, D)
    k_len = torch.tensor([Lk // 2, 0, Lk + 5], dtype=torch.int32, device="cuda")[:B] if ragged else None
    if ragged:
        for b in range(B):
            k[b, min(int(k_len[b]), Lk):] = float("nan")   # padding is never read as a value
    keys = ops().block_keys(k, k_len)
    want = ref_keys(k, k_len)
    assert bool(((keys.double() - want).abs() <= H * want.abs()).all())
    assert torch.equal(ops().block_select(q, keys, top, k_len), ref_select(q, keys, top, k_len, Lk))


@gpu
@pytest.mark.parametrize("pool", [1, 512])
def test_block_choice_ties_and_values_that_are_no_numbers(pool):
    rows_together(pool)
    g = gen(2)
    q, k = randn(g, 1, 40, 1, 16), randn(g, 1, 640, 1, 16)
    k[:, 128:192] = k[:, 448:512]            # two equal blocks
    k[:, 256:320] = 0
    k[:, 576:] = 0
    k[0, 200, 0, 3] = float("inf")
    k[0, 330, 0, 3] = float("nan")
    q[0, 0] = 0                              # every score is equal (or no number)
    q[0, 1, 0, 2] = float("nan")
    q[0, 2, 0, 3] = float("-inf")
    q[0, 3] = 1e38
    q[0, 4] *= 1e-30
    for top in (1, 2, 5, 10):
        keys = ops().block_keys(k)
        assert torch.equal(ops().block_select(q, keys, top), ref_select(q, keys, top, None, 640))


@gpu
@pytest.mark.parametrize("scale_q,scale_k", [(1.0, 1.0), (2.0 ** 40, 2.0 ** -70), (2.0 ** -80, 2.0 ** -80), (2.0 ** 60, 2.0 ** 60)])
@pytest.mark.parametrize("top", [1, 3, 8, 15, 25])
@pytest.mark.parametrize("pool", [1, 512])
def test_block_choice_among_near_ties(top, scale_q, scale_k, pool):
    """Summaries of few distinct values: many scores are equal, or differ by the last bits of a 32-bit sum."""
    rows_together(pool)
    g = gen(12)
    q = torch.randint(-3, 4, (1, 300, 2, 64), generator=g, device="cuda").to(torch.bfloat16) * scale_q
    keys = torch.randint(-2, 3, (1, 2, 130, 64), generator=g, device="cuda").to(torch.bfloat16)
    keys[:, :, ::3] += 2.0 ** -7 * torch.randint(-1, 2, (1, 2, 44, 64), generator=g, device="cuda").to(torch.bfloat16)
    keys[:, :, 5:30] *= 0     # a run of equal ones
    keys *= scale_k
    want = ref_select(q, keys, top, None, 130 * 64)
    assert torch.equal(ops().block_select(q, keys, top), want)
    assert torch.equal(ops().block_select(q[:, :7], keys, top), want[:, :, :7])


@gpu
@pytest.mark.parametrize("n,pool", [(3, 1), (40, 512)])
def test_block_choice_decides_differences_that_32_bits_cannot_hold(n, pool):
    rows_together(pool)
    # scores that differ by one part in 2^30: a large common product and a small one that differs
    q = torch.zeros(1, n, 1, 8, device="cuda", dtype=torch.bfloat16)
    q[..., 0], q[..., 1] = 1024.0, 1.0
    keys = torch.zeros(1, 1, 100, 8, device="cuda", dtype=torch.bfloat16)
    keys[..., 0] = 1024.0
    keys[0, 0, :, 1] = 2.0 ** -10 * torch.arange(100, device="cuda") * torch.where(torch.arange(100, device="cuda") % 2 == 0, 1, -1)
    got = ops().block_select(q, keys, 3)
    assert got[0, 0].tolist() == [[94, 96, 98]] * n


# -------------------------------------------------------------------------------------------------- attention
CASES = [
    # B, Lq, Lk, Hq, Hkv, D, top, ragged
    (1, 1, 1, 1, 1, 8, 1, False),
    (2, 1, 200, 4, 2, 64, 3, True),
    (1, 3, 64, 1, 1, 32, 1, False),
    (2, 63, 63, 2, 2, 16, 2, False),
    (3, 65, 129, 4, 2, 8, 2, True),
    (2, 200, 777, 6, 2, 16, 4, True),
    (1, 513, 1025, 2, 2, 32, 5, False),
    (2, 700, 1500, 4, 1, 64, 6, True),
    (1, 1100, 640, 3, 3, 64, 10, False),
    (1, 140, 5000, 2, 1, 64, 20, False),
    (4, 16, 320, 16, 16, 8, 3, False),
]


@gpu
@pytest.mark.parametrize("pool", [0, 1, 512])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,top,ragged", CASES)
def test_block_attention(B, Lq, Lk, Hq, Hkv, D, top, ragged, pool):
    rows_together(pool)
    g = gen(3)
    q, k, v, do = randn(g, B, Lq, Hq, D), randn(g, B, Lk, Hkv, D), randn(g, B, Lk, Hkv, D), randn(g, B, Lq, Hq, D)
    k_len = torch.tensor([Lk - 1, 0, Lk // 3], dtype=torch.int32, device="cuda")[:B] if ragged else None
    if ragged:
        for b in range(B):
            k[b, int(k_len[b]):], v[b, int(k_len[b]):] = float("nan"), float("inf")
    blocks = some_blocks(g, B, Hq, Lq, -(-Lk // BLOCK), top)
    scale = 1.3 * D ** -0.5
    ref = ref_attention(q, k, v, blocks, scale, k_len, do)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = ops().block_attention(*leaves, blocks, scale, k_len)
    grads = torch.autograd.grad(out, leaves, do)
    for name, got, (want, bound) in zip(("out", "dq", "dk", "dv"), (out, *grads), ref):
        within(name, got, want, bound)
    within("out without gradients", ops().block_attention(q, k, v, blocks, scale, k_len), *ref[0])


@gpu
@pytest.mark.parametrize("chosen", ["any", "one block"])
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,top,ragged", [
    (2, 700, 5000, 4, 2, 8, 12, True),
    (1, 900, 3000, 6, 3, 16, 9, False),
    (3, 333, 4111, 8, 2, 32, 7, True),
    (2, 520, 4111, 4, 1, 64, 10, True),
])
def test_block_attention_of_split_pools(B, Lq, Lk, Hq, Hkv, D, top, ragged, chosen):
    """Few pools with many blocks: the blocks are dealt to several workgroups, whose sums are joined."""
    import ctypes
    from dm_hip import lib
    g = gen(16)
    q, k, v, do = randn(g, B, Lq, Hq, D), randn(g, B, Lk, Hkv, D), randn(g, B, Lk, Hkv, D), randn(g, B, Lq, Hq, D)
    k_len = torch.tensor([Lk - 1, 0, Lk // 3], dtype=torch.int32, device="cuda")[:B] if ragged else None
    if ragged:
        for b in range(B):
            k[b, int(k_len[b]):], v[b, int(k_len[b]):] = float("nan"), float("inf")
    blocks = some_blocks(g, B, Hq, Lq, -(-Lk // BLOCK), top)
    if chosen == "one block":
        blocks.fill_(2)
    desc = ops()._block_desc(B, Lq, Lk, Hq, Hkv, D, top, 1.0, q, k, v)
    assert lib.dm_block_attention_fwd_ws_bytes(ctypes.byref(desc)) > 0
    scale = 1.3 * D ** -0.5
    ref = ref_attention(q, k, v, blocks, scale, k_len, do)

    def run(sl):
        leaves = [x[sl].clone().requires_grad_(True) for x in (q, k, v)]
        out = ops().block_attention(*leaves, blocks[sl], scale, None if k_len is None else k_len[sl])
        return [out.detach(), *torch.autograd.grad(out, leaves, do[sl])]
    got = run(slice(0, B))
    for name, x, (want, bound) in zip(("out", "dq", "dk", "dv"), got, ref):
        within(name, x, want, bound)
    within("out without gradients", ops().block_attention(q, k, v, blocks, scale, k_len), *ref[0])
    for x, y in zip(got, run(slice(B - 1, B))):   # the same bits alone
        assert torch.equal(x[B - 1:], y)


@gpu
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,top,ragged", [
    (2, 4500, 300, 2, 2, 8, 3, False),
    (3, 3000, 100, 4, 2, 16, 2, True),
    (2, 2100, 130, 4, 1, 32, 2, True),
    (1, 5000, 64, 2, 1, 64, 1, False),
])
def test_block_attention_of_few_keys_and_many_queries(B, Lq, Lk, Hq, Hkv, D, top, ragged):
    """Few blocks that many rows chose: the rows are dealt to several workgroups for dk and dv."""
    import ctypes
    from dm_hip import lib
    g = gen(18)
    q, k, v, do = randn(g, B, Lq, Hq, D), randn(g, B, Lk, Hkv, D), randn(g, B, Lk, Hkv, D), randn(g, B, Lq, Hq, D)
    k_len = torch.tensor([Lk - 1, 0, Lk // 3], dtype=torch.int32, device="cuda")[:B] if ragged else None
    if ragged:
        for b in range(B):
            k[b, int(k_len[b]):], v[b, int(k_len[b]):] = float("nan"), float("inf")
    blocks = some_blocks(g, B, Hq, Lq, -(-Lk // BLOCK), top)
    desc = ops()._block_desc(B, Lq, Lk, Hq, Hkv, D, top, 1.0, q, k, v)
    assert lib.dm_block_attention_bwd_ws_bytes(ctypes.byref(desc)) > B * Lq * Hq * 4 + 16
    scale = 1.3 * D ** -0.5
    ref = ref_attention(q, k, v, blocks, scale, k_len, do)

    def run(sl):
        leaves = [x[sl].clone().requires_grad_(True) for x in (q, k, v)]
        out = ops().block_attention(*leaves, blocks[sl], scale, None if k_len is None else k_len[sl])
        return [out.detach(), *torch.autograd.grad(out, leaves, do[sl])]
    got = run(slice(0, B))
    for name, x, (want, bound) in zip(("out", "dq", "dk", "dv"), got, ref):
        within(name, x, want, bound)
    for x, y in zip(got, run(slice(B - 1, B))):
        assert torch.equal(x[B - 1:], y)


@gpu
@pytest.mark.parametrize("pool", [1, 512])
def test_block_attention_of_one_sharp_weight(pool):
    """One key takes (almost) all the weight: ds is a small difference of large numbers."""
    rows_together(pool)
    g = gen(4)
    q, k, v, do = (randn(g, 1, 300, 2, 16) for _ in range(4))
    q *= 12
    blocks = torch.randint(0, 5, (1, 2, 300, 2), generator=g, device="cuda", dtype=torch.int32)
    ref = ref_attention(q, k, v, blocks, 0.25, None, do)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = ops().block_attention(*leaves, blocks, 0.25)
    for name, got, (want, bound) in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do)), ref):
        within(name, got, want, bound)


@gpu
@pytest.mark.parametrize("pool", [1, 512])
@pytest.mark.parametrize("scale", [-0.4, 0.0])
def test_block_attention_of_a_scale_that_is_not_positive(scale, pool):
    rows_together(pool)
    g = gen(13)
    q, k, v, do = randn(g, 1, 90, 2, 16), randn(g, 1, 150, 1, 16), randn(g, 1, 150, 1, 16), randn(g, 1, 90, 2, 16)
    blocks = some_blocks(g, 1, 2, 90, 3, 2)
    ref = ref_attention(q, k, v, blocks, scale, None, do)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    out = ops().block_attention(*leaves, blocks, scale)
    for name, got, (want, bound) in zip(("out", "dq", "dk", "dv"), (out, *torch.autograd.grad(out, leaves, do)), ref):
        within(name, got, want, bound)


@gpu
def test_block_attention_gradient_against_differences():
    g = gen(5)
    q, k, v, do = randn(g, 1, 70, 2, 16), randn(g, 1, 150, 1, 16), randn(g, 1, 150, 1, 16), randn(g, 1, 70, 2, 16)
    blocks = some_blocks(g, 1, 2, 70, 3, 2)
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]
    grads = torch.autograd.grad(ops().block_attention(*leaves, blocks, 0.25), leaves, do)
    # central differences of the 64-bit definition along random directions, h^2 error below 2^-12 of the slope
    for x, got in enumerate(grads):
        u = torch.randn(leaves[x].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 2.0 ** -9
        side = []
        for sign in (1, -1):
            moved = [t.double() for t in (q, k, v)]
            moved[x] = moved[x] + sign * h * u
            side.append((ref_attention(*moved, blocks, 0.25, None, do)[0][0] * do.double()).sum())
        slope = float((side[0] - side[1]) / (2 * h))
        bound = ref_attention(q, k, v, blocks, 0.25, None, do)[x + 1][1]
        assert abs(float((got.double() * u).sum()) - slope) <= float((bound * u.abs()).sum()) + 2.0 ** -10 * abs(slope)


@gpu
def test_block_attention_reads_strided_tensors_in_place_and_copies_others():
    g = gen(6)
    B, L, Hh, D = 2, 150, 3, 16
    qkv = randn(g, B, L, 3, Hh, D)
    q, k, v = qkv.unbind(2)
    blocks = some_blocks(g, B, Hh, L, 3, 2)
    want = ops().block_attention(q.contiguous(), k.contiguous(), v.contiguous(), blocks)
    assert torch.equal(ops().block_attention(q, k, v, blocks), want)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(ops().block_attention(*heads_first, blocks), want)
    odd = torch.empty(B * L * Hh * D + 1, device="cuda", dtype=torch.bfloat16)[1:].view(B, L, Hh, D)   # rows off 16 bytes
    assert torch.equal(ops().block_attention(q, odd.copy_(k), v, blocks), want)
    assert torch.equal(ops().block_attention(q.float(), k.float(), v.float(), blocks), want)
    # one value for every head and position: its gradient is the sum over both
    one = randn(g, B, 1, 1, D).requires_grad_(True)
    full = one.detach().expand(B, L, Hh, D).clone().requires_grad_(True)
    do = randn(g, B, L, Hh, D)
    a, = torch.autograd.grad(ops().block_attention(q, k, one.expand(B, L, Hh, D), blocks), one, do)
    b, = torch.autograd.grad(ops().block_attention(q, k, full, blocks), full, do)
    assert torch.equal(a, b.sum((1, 2), keepdim=True)) or rel_err(a.float().cpu(), b.float().sum((1, 2), keepdim=True).cpu()) < 2 * H


@gpu
@pytest.mark.parametrize("B,Lq,Lk", [(0, 3, 70), (2, 0, 70), (2, 3, 0)])
def test_block_attention_of_nothing(B, Lq, Lk):
    mk = lambda L: torch.full((B, L, 2, 16), float("nan"), device="cuda", dtype=torch.bfloat16, requires_grad=True)  # noqa: E731
    q, k, v = mk(Lq), mk(Lk), mk(Lk)
    blocks = torch.zeros(B, 2, Lq, 3, dtype=torch.int32, device="cuda")
    out = ops().block_attention(q, k, v, blocks)
    assert out.shape == q.shape and not bool(out.any())
    for g_, x in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
        assert g_.shape == x.shape and not bool(g_.any())
    keys = ops().block_keys(k)
    assert keys.shape == (B, 2, -(-Lk // 64), 16)
    picked = ops().block_select(q, keys, 3)
    assert picked.shape == (B, 2, Lq, 3) and bool((picked == -1).all() or Lk)


@gpu
@pytest.mark.parametrize("B,L,Hh,D,top", [(2, 130, 4, 8, 1), (1, 1024, 2, 64, 4), (3, 64, 5, 16, 2), (2, 1, 2, 32, 1)])
def test_sparse_attention_packed(B, L, Hh, D, top):
    g = gen(7)
    qkv = randn(g, B, L, 3 * Hh * D)
    do = randn(g, B, L, Hh * D)
    q, k, v = qkv.view(B, L, 3, Hh, D).unbind(2)
    blocks = ops().block_select(q, ops().block_keys(k), top)
    assert torch.equal(blocks, ref_select(q, ops().block_keys(k), top, None, L))
    leaf = qkv.clone().requires_grad_(True)
    out = ops().sparse_attention(leaf, Hh, D, top)
    (dqkv,) = torch.autograd.grad(out, leaf, do)
    ref = ref_attention(q, k, v, blocks, D ** -0.5, None, do.view(B, L, Hh, D))
    parts = dqkv.view(B, L, 3, Hh, D).unbind(2)
    for name, got, (want, bound) in zip(("out", "dq", "dk", "dv"), (out.view(B, L, Hh, D), *parts), ref):
        within(name, got, want, bound)
    if top * 64 >= L:   # every block: the dense operator's result, both rounded
        dense = ops().attention(qkv, Hh, D).view(B, L, Hh, D)
        within("dense", dense, *(ref[0][0], 2 * ref[0][1]))


@gpu
def test_block_attention_same_bits_whatever_the_batch():
    g = gen(8)
    q, k, v, do = (randn(g, 3, 600, 4, 64) for _ in range(4))
    blocks = some_blocks(g, 3, 4, 600, 10, 3)

    def run(sl):
        leaves = [x[sl].clone().requires_grad_(True) for x in (q, k, v)]
        out = ops().block_attention(*leaves, blocks[sl])
        return [out.detach(), *torch.autograd.grad(out, leaves, do[sl])]
    whole = run(slice(0, 3))
    for a, b in zip(whole, run(slice(0, 3))):
        assert torch.equal(a, b)
    for a, b in zip(whole, run(slice(1, 2))):
        assert torch.equal(a[1:2], b)


# -------------------------------------------------------------------------------------------------- embedding
@gpu
@pytest.mark.parametrize("n,rows,width,padding,out,scale", [
    (1, 1, 1, None, "float32", 1.0),
    (3, 5, 7, 4, "bfloat16", 3.0),
    (256, 11, 512, 10, "float32", 1.0),
    (1000, 300, 33, -1, "float32", 0.5),
    (2048, 256, 20, None, "bfloat16", 1.0),
    (2049, 257, 64, 0, "float32", -2.0),
    (5000, 70000, 12, 3, "bfloat16", 1.0),      # three sort passes
    (8192, 3000, 8, None, "float32", 1.0),      # the largest call that one workgroup sorts
    (8193, 70000, 8, 2, "float32", 1.0),        # ... and the smallest that it does not
    (526000, 700, 8, None, "float32", 1.0),     # so many tiles that their counts are summed by themselves
    (1100000, 300000, 2, 3, "bfloat16", 1.0),   # ... in three passes
    (9000, 2 ** 24 + 5, 4, 2, "float32", 1.0),  # four passes
    (30000, 2, 8, None, "float32", 1.0),        # two runs over nearly every chunk
    (66000, 3, 1, None, "bfloat16", 1.0),       # one feature; long chunks and joins of many parts
    (3000, 5000, 2, 7, "float32", 1.0),
    (40000, 33, 1024, 5, "float32", 1.0),       # four rows a thread
    (70000, 900, 260, 1, "bfloat16", 22.0),     # the longer chunks of large calls
    (400, 50, 1500, None, "float32", 1.0),      # more features than one workgroup takes
])
def test_token_embed(n, rows, width, padding, out, scale):
    g = gen(9)
    dtype = getattr(torch, out)
    table = torch.randn(rows, width, generator=g, device="cuda")
    tokens = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) ** 3 * rows).long().clamp(max=rows - 1)
    if n > 100:
        tokens[::17] = -1          # no tokens of the table
        tokens[5::29] = rows
        tokens[7] = 2 ** 40
    ok = (tokens >= 0) & (tokens < rows)
    leaf = table.clone().requires_grad_(True)
    got = ops().token_embed(tokens, leaf, scale, padding, dtype)
    half = H if dtype == torch.bfloat16 else 2.0 ** -24
    want = torch.where(ok[:, None], table.double()[tokens.clamp(0, rows - 1)] * scale, 0.0)
    assert got.dtype == dtype and bool(((got.double() - want).abs() <= 2 * 2.0 ** -24 * want.abs() + half * want.abs()).all())
    assert torch.equal(got, ops().token_embed(tokens, table, scale, padding, dtype))
    dout = torch.randn(n, width, generator=g, device="cuda").to(dtype)
    (grad,) = torch.autograd.grad(got, leaf, dout)
    pad = None if padding is None else padding % rows
    keep = ok if pad is None else ok & (tokens != pad)
    term = dout.double()[keep] * scale
    ref = torch.zeros(rows, width, dtype=torch.float64, device="cuda").index_add_(0, tokens[keep], term)
    size = torch.zeros_like(ref).index_add_(0, tokens[keep], term.abs())
    count = torch.zeros(rows, dtype=torch.float64, device="cuda").index_add_(0, tokens[keep], torch.ones_like(tokens[keep], dtype=torch.float64))
    assert bool(((grad.double() - ref).abs() <= (count[:, None] + 2) * 2.0 ** -24 * size).all())
    (again,) = torch.autograd.grad(ops().token_embed(tokens, leaf, scale, padding, dtype), leaf, dout)
    assert torch.equal(grad, again)


@gpu
def test_token_embed_shapes_types_and_an_empty_call():
    g = gen(10)
    table = torch.randn(9, 6, generator=g, device="cuda", requires_grad=True)
    t = torch.randint(0, 9, (4, 5), generator=g, device="cuda", dtype=torch.int32)
    out = ops().token_embed(t.t(), table, dtype=torch.float32)
    assert torch.equal(out, table.detach()[t.t().long()])
    out.backward(torch.ones_like(out))
    assert torch.equal(table.grad.sum(1), 6.0 * torch.bincount(t.flatten().long(), minlength=9))
    none = ops().token_embed(torch.empty(0, 3, dtype=torch.int64, device="cuda"), table)
    assert none.shape == (0, 3, 6) and not bool(torch.autograd.grad(none, table, torch.empty_like(none))[0].any())
    half = table.detach().to(torch.bfloat16).requires_grad_(True)
    (gr,) = torch.autograd.grad(ops().token_embed(t, half), half, torch.ones(4, 5, 6, device="cuda", dtype=torch.bfloat16))
    assert gr.dtype == torch.bfloat16
    at_odd = torch.randn(9 * 6 + 1, generator=g, device="cuda")[1:].view(9, 6)   # 4-byte aligned rows
    assert torch.equal(ops().token_embed(t, at_odd, dtype=torch.float32), at_odd[t.long()])


@gpu
def test_token_embed_gradient_accumulates_into_the_arena():
    o = ops()
    g = gen(11)
    table = torch.nn.Parameter(torch.randn(20, 8, generator=g, device="cuda"))
    t = torch.randint(0, 20, (100,), generator=g, device="cuda")
    dout = torch.randn(100, 8, generator=g, device="cuda")
    (want,) = torch.autograd.grad(o.token_embed(t, table, dtype=torch.float32), table, dout)
    table.grad = torch.ones_like(table)
    ready = []
    o.DIRECT_GRADS, o.GRAD_READY = True, ready.append
    try:
        o.token_embed(t, table, dtype=torch.float32).backward(dout)
    finally:
        o.DIRECT_GRADS, o.GRAD_READY = False, None
    assert len(ready) == 1 and ready[0] is table
    assert bool(((table.grad - 1 - want).abs() <= 2.0 ** -23 * (1 + want.abs())).all())


# -------------------------------------------------------------------------------------------------- refusals (no GPU needed)
def test_refusals_of_tensors_on_the_cpu():
    o = ops()
    x, t = torch.zeros(1, 2, 1, 8, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: o.block_keys(x), lambda: o.block_select(x, x, 1), lambda: o.sparse_attention(x[:, :, 0], 1, 8, 1),
                 lambda: o.block_attention(x, x, x, torch.zeros(1, 1, 2, 1, dtype=torch.int32)), lambda: o.token_embed(t, torch.zeros(3, 4))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()


def test_refusals_of_the_c_abi():
    """Argument checks come before anything touches the device, and report through dm_last_error."""
    from dm_hip import BlockDesc, lib
    p = ctypes.c_void_p(4096)

    def desc(**kw):
        d = BlockDesc(1, 64, 64, 2, 1, 16, 4, 0, 1.0)
        for s in ("q_stride", "k_stride", "v_stride", "dq_stride", "dk_stride", "dv_stride"):
            getattr(d, s)[:] = [2048, 32, 16]
        for k, v in kw.items():
            if isinstance(v, list):
                getattr(d, k)[:] = v
            else:
                setattr(d, k, v)
        return ctypes.byref(d)

    for kw, code, text in [(dict(D=24), 2, "head dim"), (dict(D=128), 2, "head dim"), (dict(top=0), 2, "top"), (dict(top=65), 2, "top"),
                           (dict(Hq=3, Hkv=2), 2, "evenly"), (dict(Lk=0), 2, "positive"), (dict(B=-1), 2, "positive"),
                           (dict(B=70000), 2, "65535"), (dict(k_stride=[2048, 36, 16]), 1, "multiples of 8")]:
        assert lib.dm_block_keys(desc(**kw), p, None, p, None) == code
        assert text in lib.dm_last_error().decode()
    assert lib.dm_block_keys(None, p, None, p, None) == 1
    assert lib.dm_block_keys(desc(), None, None, p, None) == 1
    assert lib.dm_block_keys(desc(), ctypes.c_void_p(4100), None, p, None) == 1
    assert lib.dm_block_select(desc(q_stride=[2048, 33, 16]), p, p, None, p, None) == 1
    assert lib.dm_block_select(desc(), p, p, None, None, None) == 1
    assert lib.dm_block_attention_fwd(desc(), p, p, p, None, None, p, None, None, None, None, 0, None) == 1
    assert lib.dm_block_attention_fwd(desc(pool=512), p, p, p, p, None, p, None, None, None, None, 0, None) == 1
    assert "plan" in lib.dm_last_error().decode()
    assert lib.dm_block_attention_bwd(desc(), p, p, p, p, None, p, p, p, p, p, p, p, p, p, 8, None) == 1
    assert "workspace" in lib.dm_last_error().decode()
    assert lib.dm_block_attention_plan_bytes(desc(D=3), 1) == 0
    assert lib.dm_block_attention_plan_bytes(desc(pool=64), 1) == 0
    assert lib.dm_block_attention_fwd(desc(q_stride=[0, 2 ** 32, 16]), p, p, p, p, None, p, None, None, p, None, 0, None) == 2
    assert lib.dm_token_embed(p, p, p, 0, 5, 0, 4, 1.0, None) == 2
    assert lib.dm_token_embed(p, p, p, 0, 2 ** 31, 9, 4, 1.0, None) == 2
    assert lib.dm_token_embed(p, p, p, 0, 5, 9, 0, 1.0, None) == 2
    assert lib.dm_token_embed(p, None, p, 0, 5, 9, 4, 1.0, None) == 1
    assert lib.dm_token_embed(None, None, None, 0, 0, 9, 4, 1.0, None) == 0
    assert lib.dm_token_embed_bwd(p, 0, p, p, 5, 9, 4, 1.0, -1, 1, p, 16, None) == 1
    assert lib.dm_token_embed_bwd_ws_bytes(5, 9, -1) == 0


@gpu
def test_refusals():
    o = ops()
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.bfloat16)          # noqa: E731
    i = lambda *s: torch.zeros(*s, device="cuda", dtype=torch.int32)             # noqa: E731
    q, k = z(2, 5, 4, 16), z(2, 70, 2, 16)
    good = i(2, 4, 5, 3)
    o.block_attention(q, k, k, good)
    for bad in [lambda: o.block_attention(q[0], k, k, good), lambda: o.block_attention(z(2, 5, 4, 24), z(2, 70, 2, 24), z(2, 70, 2, 24), good),
                lambda: o.block_attention(q, z(1, 70, 2, 16), z(1, 70, 2, 16), good), lambda: o.block_attention(q, k, z(2, 71, 2, 16), good),
                lambda: o.block_attention(q, z(2, 70, 3, 16), z(2, 70, 3, 16), good), lambda: o.block_attention(q, k, k, good.long()),
                lambda: o.block_attention(q, k, k, i(2, 5, 4, 3)), lambda: o.block_attention(q, k, k, i(2, 4, 5, 65)),
                lambda: o.block_attention(q, k, k, i(2, 4, 5, 0)), lambda: o.block_attention(q, k, k, good.cpu()),
                lambda: o.block_attention(q, k, k, good, k_len=torch.ones(2, device="cuda")),
                lambda: o.block_attention(q, k, k, good, k_len=i(3)), lambda: o.block_attention(q, k, k, good, k_len=torch.ones(2, dtype=torch.int32)),
                lambda: o.block_select(q, z(2, 3, 2, 16), 2), lambda: o.block_select(q, z(2, 2, 2, 8), 2), lambda: o.block_select(q, o.block_keys(k), 0),
                lambda: o.sparse_attention(z(2, 5, 48), 2, 16, 1), lambda: o.sparse_attention(z(2, 5, 72), 1, 24, 1),
                lambda: o.sparse_attention(z(2, 5, 48), 1, 16, 65),
                lambda: o.token_embed(torch.zeros(3, device="cuda"), torch.zeros(3, 4, device="cuda")),
                lambda: o.token_embed(i(3), torch.zeros(12, device="cuda")), lambda: o.token_embed(i(3), torch.zeros(3, 4, device="cuda"), dtype=torch.float16),
                lambda: o.token_embed(i(3), torch.zeros(3, 4, device="cuda"), padding_idx=3), lambda: o.token_embed(i(3).cpu(), torch.zeros(3, 4, device="cuda"))]:
        with pytest.raises(RuntimeError):
            bad()


# -------------------------------------------------------------------------------------------------- streams, graphs, long offsets
def _everything(x):
    """one pass through every operator; x: the inputs, returned: every result"""
    o = ops()
    emb = o.token_embed(x["tokens"], x["table"], 1.5, 0, torch.float32)
    grads = list(torch.autograd.grad(emb, x["table"], x["demb"]))
    keys = o.block_keys(x["k"].detach(), x["k_len"])
    blocks = o.block_select(x["q"].detach(), keys, 3, x["k_len"])
    att = o.block_attention(x["q"], x["k"], x["v"], blocks, k_len=x["k_len"])
    grads += torch.autograd.grad(att, (x["q"], x["k"], x["v"]), x["datt"])
    packed = o.sparse_attention(x["qkv"], 4, 16, 2)
    grads += torch.autograd.grad(packed, x["qkv"], x["dpacked"])
    return [emb.detach(), keys, blocks, att.detach(), packed.detach()] + grads


def _inputs(seed):
    g = gen(seed)
    x = {"table": torch.randn(50, 24, generator=g, device="cuda"), "q": randn(g, 2, 600, 4, 16), "k": randn(g, 2, 700, 2, 16),
         "v": randn(g, 2, 700, 2, 16), "qkv": randn(g, 2, 520, 3 * 64)}
    x = {n: t.requires_grad_(True) for n, t in x.items()}
    x["k_len"] = torch.tensor([seed * 37 % 701, 700], dtype=torch.int32, device="cuda")
    x["tokens"] = torch.randint(0, 50, (9000,), generator=g, device="cuda")
    x["demb"], x["datt"], x["dpacked"] = torch.randn(9000, 24, generator=g, device="cuda"), randn(g, 2, 600, 4, 16), randn(g, 2, 520, 64)
    return x


@gpu
@pytest.mark.parametrize("pool", [0, 1, 512])
def test_graph_replays_equal_eager(pool):
    rows_together(pool)
    want = [[t.clone() for t in _everything(_inputs(s))] for s in (1, 2, 3)]   # (the eager graphs are gone before the capture)
    static = _inputs(1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _everything(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = ops().new_graph()
    with torch.cuda.graph(graph):
        got = _everything(static)
    for s in (1, 2, 3, 2, 1):
        fresh = _inputs(s)
        with torch.no_grad():
            for n in static:
                static[n].copy_(fresh[n])
        graph.replay()
        for a, b in zip(got, want[s - 1]):
            assert torch.equal(a, b)
        torch.randn(1 << 20, device="cuda").sum().item()      # eager work between the replays


@gpu
def test_two_captured_graphs_do_not_share_scratch():
    a, b = _inputs(4), _inputs(5)
    want = [[t.clone() for t in _everything(x)] for x in (_inputs(4), _inputs(5))]
    graphs, got = [], []
    for x in (a, b):
        g = ops().new_graph()
        with torch.cuda.graph(g):
            got.append(_everything(x))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for g, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                g.replay()
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        for res, ref in zip(got, want):
            for u, v in zip(res, ref):
                assert torch.equal(u, v)


@gpu
def test_graph_of_split_pools():
    def inputs(seed):
        g = gen(seed)
        x = {"q": randn(g, 3, 333, 8, 32), "k": randn(g, 3, 4111, 2, 32), "v": randn(g, 3, 4111, 2, 32)}
        x = {n: t.requires_grad_(True) for n, t in x.items()}
        x["blocks"], x["do"] = some_blocks(g, 3, 8, 333, 65, 7), randn(g, 3, 333, 8, 32)
        return x

    def step(x):
        leaves = [x[n] for n in "qkv"]
        out = ops().block_attention(*leaves, x["blocks"])
        return [out.detach(), *torch.autograd.grad(out, leaves, x["do"])]
    want = [[t.clone() for t in step(inputs(s))] for s in (1, 2)]
    static = inputs(1)
    graph = ops().new_graph()
    with torch.cuda.graph(graph):
        got = step(static)
    for s in (2, 1, 2):
        fresh = inputs(s)
        with torch.no_grad():
            for n in static:
                static[n].copy_(fresh[n])
        graph.replay()
        for a, b in zip(got, want[s - 1]):
            assert torch.equal(a, b)
        torch.randn(1 << 20, device="cuda").sum().item()


@gpu
def test_more_workgroups_than_one_dimension_holds():
    """Over 2^20 workgroups: queries taken one by one, and token rows. The end of the call equals a call for the end."""
    rows_together(1)
    g = gen(17)
    L, tail = (1 << 22) + 4099, 5000
    q, k, v, do = randn(g, 1, L, 1, 8), randn(g, 1, 130, 1, 8), randn(g, 1, 130, 1, 8), randn(g, 1, L, 1, 8)
    keys = ops().block_keys(k)
    blocks = ops().block_select(q, keys, 2)
    end = slice(L - tail, L)
    assert torch.equal(blocks[:, :, end], ops().block_select(q[:, end], keys, 2))
    leaf, part = q.requires_grad_(True), q[:, end].detach().clone().requires_grad_(True)
    out = ops().block_attention(leaf, k, v, blocks)
    small = ops().block_attention(part, k, v, blocks[:, :, end])
    assert torch.equal(out[:, end], small)
    (dq,), (dp,) = torch.autograd.grad(out, leaf, do), torch.autograd.grad(small, part, do[:, end])
    assert torch.equal(dq[:, end], dp)
    table = torch.randn(3, 257, generator=g, device="cuda")
    tokens = torch.randint(0, 3, (L,), generator=g, device="cuda")
    rows = ops().token_embed(tokens, table)
    assert torch.equal(rows[-tail:], table[tokens[-tail:]].to(torch.bfloat16)) and torch.equal(rows[:tail], table[tokens[:tail]].to(torch.bfloat16))


@gpu
def test_saved_tensors_that_come_back_from_elsewhere():
    g = gen(19)
    q, k, v, do = (randn(g, 2, 130, 4, 16) for _ in range(4))
    blocks = some_blocks(g, 2, 4, 130, 3, 2)
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    want = torch.autograd.grad(ops().block_attention(*leaves, blocks), leaves, do)

    def heads_first(t):   # the same values, laid out otherwise
        t = t.cuda()
        return t.transpose(1, 2).contiguous().transpose(1, 2) if t.shape == q.shape and any(torch.equal(t, x) for x in leaves) else t
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), heads_first):
        out = ops().block_attention(*leaves, blocks)
    for a, b in zip(torch.autograd.grad(out, leaves, do), want):
        assert torch.equal(a, b)
    qkv, dp = randn(g, 2, 260, 3 * 64).requires_grad_(True), randn(g, 2, 260, 64)
    want = torch.autograd.grad(ops().sparse_attention(qkv, 4, 16, 2), qkv, dp)
    with torch.autograd.graph.save_on_cpu():
        out = ops().sparse_attention(qkv, 4, 16, 2)
    assert torch.equal(torch.autograd.grad(out, qkv, dp)[0], want[0])


@gpu
def test_on_a_stream_of_the_callers():
    want = _everything(_inputs(6))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = _inputs(6)
        got = _everything(x)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("pool", [1, 512])
def test_offsets_beyond_32_bits(pool):
    """A sequence whose keys are 2^31 elements and more (4.4 GB), attended to at its end, equals the end by itself."""
    rows_together(pool)
    g = gen(14)
    L, tail = 4_300_000 // 64 * 64, 64 * 40
    k = torch.zeros(1, L + 17, 8, 64, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    assert k.numel() > 2 ** 31
    k[:, L - tail:], v[:, L - tail:] = randn(g, 1, tail + 17, 8, 64), randn(g, 1, tail + 17, 8, 64)
    ke, ve = k[:, L - tail:].clone(), v[:, L - tail:].clone()
    first = (L - tail) // 64
    for Lq in (2, 600):
        q = randn(g, 1, Lq, 8, 64, scale=2.0)
        keys = ops().block_keys(k)
        assert torch.equal(keys[:, :, first:], ops().block_keys(ke)) and not bool(keys[:, :, :first].any())
        blocks = ops().block_select(q, keys, 4)
        near = ops().block_select(q, keys[:, :, first:], 4)
        assert torch.equal(blocks, near + first)   # a summary of zero never beats the best of 40 random ones here
        assert torch.equal(ops().block_attention(q, k, v, blocks), ops().block_attention(q, ke, ve, near))
    leaves = [x.requires_grad_(True) for x in (q, k, v)]
    small = [x.detach().clone().requires_grad_(True) for x in (q, ke, ve)]
    do = randn(g, 1, 600, 8, 64)
    dq, dk, dv = torch.autograd.grad(ops().block_attention(*leaves, blocks), leaves, do)
    sq, sk, sv = torch.autograd.grad(ops().block_attention(*small, near), small, do)
    assert torch.equal(dq, sq) and torch.equal(dk[:, L - tail:], sk) and torch.equal(dv[:, L - tail:], sv)
    assert not bool(dk[:, :L - tail].any())


@gpu
def test_token_embed_offsets_beyond_32_bits():
    rows, width = 70000, 32768
    table = torch.zeros(rows, width, device="cuda")
    assert table.numel() > 2 ** 31
    table[rows - 3:] = torch.randn(3, width, generator=gen(15), device="cuda")
    tokens = torch.tensor([rows - 1, 0, rows - 3, rows - 1], device="cuda")
    leaf = table.requires_grad_(True)
    out = ops().token_embed(tokens, leaf, dtype=torch.float32)
    assert torch.equal(out, table.detach()[tokens])
    (grad,) = torch.autograd.grad(out, leaf, torch.ones_like(out))
    assert grad[rows - 1].eq(2).all() and grad[rows - 3].eq(1).all() and grad[0].eq(1).all() and float(grad.sum()) == 4.0 * width


# -------------------------------------------------------------------------------------------------- in the model
def test_attention_layer_keeps_its_parameters_and_refuses():
    from modeling.attention import Attention2D
    from modeling.unet import UNet
    assert list(Attention2D(64, n_dim_head=8).state_dict()) == list(Attention2D(64, n_dim_head=8, top_blocks=3).state_dict())
    assert Attention2D(64, n_dim_head=8, n_context=128).context_proj.weight.shape == (128, 128)
    for bad in (lambda: Attention2D(64, n_dim_head=8, top_blocks=0), lambda: Attention2D(64, n_dim_head=8, top_blocks=65),
                lambda: Attention2D(64, n_dim_head=8, top_blocks=2, dropout=0.1), lambda: Attention2D(64, n_dim_head=8, n_context=63),
                lambda: Attention2D(64, n_dim_head=8, n_context=64, dropout=0.1)):
        with pytest.raises(ValueError):
            bad()
    net = UNet(block_out_channels=(64, 64), down_block_types=("UNetDownBlock", "UNetAttnDownBlock"),
               up_block_types=("UNetAttnUpBlock", "UNetUpBlock"), n_dim_attention_head=8, attention_top_blocks=2)
    layers = [m for m in net.modules() if isinstance(m, Attention2D)]
    assert layers and all(m.top_blocks == 2 for m in layers)


def _layer(seed, **kw):
    from modeling.attention import Attention2D
    torch.manual_seed(seed)
    return Attention2D(64, n_dim_head=8, norm_groups=8, **kw).cuda()


def _plain_layer(m, x, blocks_of, context=None, context_len=None):
    """the layer in fp32 from its parameters, attending where `blocks_of(q, k)` says"""
    B, C, Hh, W = x.shape
    L = Hh * W
    h = torch.nn.functional.group_norm(x, m.norm.num_groups, m.norm.weight, m.norm.bias, m.norm.eps)
    qkv = torch.nn.functional.linear(h.flatten(2).transpose(1, 2), m.qkv_proj.weight, m.qkv_proj.bias)
    q, k, v = qkv.view(B, L, 3, m.n_heads, m.n_dim_head).unbind(2)
    live = torch.ones(B, L, dtype=torch.bool, device="cuda")
    if context is not None:
        kv = torch.nn.functional.linear(context, m.context_proj.weight, m.context_proj.bias)
        T = context.shape[1]
        ck, cv = kv.view(B, T, 2, m.n_heads, m.n_dim_head).unbind(2)
        k, v = torch.cat([k, ck], 1), torch.cat([v, cv], 1)
        live = torch.cat([live, torch.arange(T, device="cuda") < context_len[:, None]], 1)
    Lk = k.shape[1]
    picked = blocks_of(q, k, live)
    s = torch.matmul(q.transpose(1, 2), k.transpose(1, 2).transpose(2, 3)) * m.n_dim_head ** -0.5
    s = s.masked_fill(~(picked.repeat_interleave(64, 3)[..., :Lk] & live[:, None, None]), -float("inf"))
    att = torch.matmul(torch.softmax(s, -1), v.transpose(1, 2)).transpose(1, 2).reshape(B, L, -1)
    out = torch.nn.functional.linear(att, m.out_proj.weight, m.out_proj.bias)
    return x + out.transpose(1, 2).view(B, C, Hh, W)


@gpu
def test_attention_layer_on_chosen_blocks(monkeypatch):
    o = ops()
    m = _layer(1, top_blocks=2)
    g = gen(16)
    x = torch.randn(2, 64, 20, 18, generator=g, device="cuda").to(torch.bfloat16).float()     # 360 pixels: 6 blocks
    do = torch.randn(2, 64, 20, 18, generator=g, device="cuda").to(torch.bfloat16)
    made, select = [], o.block_select
    monkeypatch.setattr(o, "block_select", lambda *a, **k: made.append(select(*a, **k)) or made[-1])
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    out = m(b)
    got = torch.autograd.grad(out, [b, *m.parameters()], do)
    assert len(made) == 1
    picked = torch.zeros(2, m.n_heads, 360, 6, dtype=torch.bool, device="cuda").scatter_(3, made[0].long(), True)
    ref = _plain_layer(m, a, lambda q, k, live: picked)     # (the choice itself is tested by itself: it has no gradient)
    want = torch.autograd.grad(ref, [a, *m.parameters()], do.float())
    # a handful of bf16 roundings (2^-8 each) one behind the other, as for the dense layer
    assert rel_err(out.detach().float().cpu(), ref.detach().cpu()) < 1e-2
    for u, v in zip(got, want):
        assert rel_err(u.float().cpu(), v.cpu()) < 3e-2
    m.attend_to(6)             # as many blocks as there are: the dense operator
    assert torch.equal(m(b), _layer(1)(b)) and len(made) == 1


@gpu
def test_text_conditioned_attention_from_tokens_to_their_table():
    """Token rows -> keys and values beside the pixels' -> attention of pixels over both -> gradients back into the rows."""
    from modeling.layers import TokenEmbedding
    torch.manual_seed(3)
    emb = TokenEmbedding(40, 128, padding_idx=0, scale=128 ** 0.5 / 8).cuda()
    m = _layer(2, n_context=128)
    g = gen(19)
    tokens = torch.randint(1, 40, (3, 20), generator=g, device="cuda")
    length = torch.tensor([20, 0, 7], device="cuda")
    tokens[torch.arange(20, device="cuda") >= length[:, None]] = 0
    x = torch.randn(3, 64, 9, 9, generator=g, device="cuda").to(torch.bfloat16).float()
    do = torch.randn(3, 64, 9, 9, generator=g, device="cuda").to(torch.bfloat16)
    a, b = x.clone().requires_grad_(True), x.clone().requires_grad_(True)
    params = [emb.weight, *m.parameters()]
    every = lambda q, k, live: torch.ones(3, m.n_heads, q.shape[1], -(-k.shape[1] // 64), dtype=torch.bool, device="cuda")  # noqa: E731
    ref = _plain_layer(m, a, every, emb.weight[tokens] * emb.scale, length)
    want = torch.autograd.grad(ref, [a, *params], do.float())
    out = m(b, context=emb(tokens), context_len=length)
    got = torch.autograd.grad(out, [b, *params], do)
    assert rel_err(out.detach().float().cpu(), ref.detach().cpu()) < 1e-2
    for u, v in zip(got, want):
        assert rel_err(u.float().cpu(), v.float().cpu()) < 3e-2
    assert not bool(got[1][0].any())                   # the padding row
    # the padded text changes nothing, the valid one does
    other = tokens.clone()
    other[2, 7:] = 5
    assert torch.equal(m(b, context=emb(other), context_len=length), out)
    m.attend_to(1)
    assert m(b, context=emb(tokens), context_len=length).shape == out.shape
    with pytest.raises(RuntimeError):
        m(b, context=emb(tokens)[:2])
    with pytest.raises(RuntimeError):
        _layer(2)(b, context=emb(tokens))


@gpu
def test_unet_attending_to_chosen_blocks():
    from modeling.unet import UNet
    kw = dict(block_out_channels=(64, 64), down_block_types=("UNetAttnDownBlock", "UNetDownBlock"),
              up_block_types=("UNetUpBlock", "UNetAttnUpBlock"), n_blocks_per_layer=1, n_dim_attention_head=8, norm_groups=8,
              time_encoding_dim=64, embedding_dim=64)
    nets = []
    for top in (None, 16, 3):
        torch.manual_seed(4)
        nets.append(UNet(attention_top_blocks=top, **kw).cuda())
    g = gen(20)
    x, t = torch.randn(4, 3, 32, 32, generator=g, device="cuda"), torch.randint(0, 1000, (4,), generator=g, device="cuda")
    with torch.no_grad():
        dense, full, sparse = (n(x, t) for n in nets)
        assert torch.equal(dense, full)                # 32x32 pixels are 16 blocks
        assert not torch.equal(dense, sparse)
        assert torch.equal(nets[2](x[1:3], t[1:3]), sparse[1:3])   # whatever the batch
    nets[2](x, t).square().mean().backward()
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in nets[2].parameters())
