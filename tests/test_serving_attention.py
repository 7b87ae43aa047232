"""Cross attention with padding and shared K/V heads, and attention over a prefix that a batch shares
(`attention.cross_attention`, `attention.prefix_attention`), against float64."""
import math

import pytest
import torch

from conftest import seeded

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def heads(g, dtype, *shape):
    return torch.randn(*shape, generator=g).to(dtype)


def attend64(q, k, v, seen, scale, coded=None):
    """q [Lq, D], k / v [n, D] float64, seen [Lq, n] -> (result, sum of p |v| / sum of p, sum of |v| / sum of p, score size).
    `coded`: (codes, scales) of the first values; they enter the third sum as |code| times the row's largest p * scale."""
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z, z, torch.zeros(q.shape[0], 1, dtype=q.dtype, device=q.device)
    s = (q @ k.t().contiguous()) * scale
    s = torch.where(seen, s, -math.inf)
    top = s.amax(1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(top.isinf(), 0.0, top)), 0.0)
    total = p.sum(1, keepdim=True)
    total = torch.where(total > 0, total, 1.0)
    vs = v.abs()
    size = (q.abs() @ k.abs().t().contiguous() * scale * seen).amax(1, keepdim=True)
    flat = seen.double() @ vs
    if coded is not None and coded[0].shape[0]:
        c, at = coded[0].shape[0], coded[0].double().abs()
        flat = seen[:, :c].double() @ at * (p[:, :c] * coded[1].double()).amax(1, keepdim=True) + seen[:, c:].double() @ vs[c:]
    return p @ v / total, p @ vs / total, flat / total, size


def check(got, q, rows, coded=None):
    """`rows(b, h)` -> (k, v, seen, scale) of one sample and query head in float64.  Each element is off by at most: half a step of the
    type for its own rounding; half a step of the type for each probability (relative, so of sum p |v|; fp16 ones below
    2^-14 are off by 2^-25 instead); the error of the scores, D + 8 half steps of fp32 of the largest sum |q k|, twice (in the
    numerator and the sum); n + 64 half steps of fp32 for the sums over n keys, their rescaling and the exponentials.
    `coded(h)`: codes and scales of the first values.  What is rounded for them is the probability times the scale: fp16 ones below
    2^-14 of the row's largest are off by 2^-25 of that, for each code."""
    b, lq, hq, d = q.shape
    u = torch.finfo(q.dtype).eps / 2
    worst = 0.0
    for i in range(b):
        for h in range(hq):
            k, v, seen, scale = rows(i, h)
            ref, mag, flat, size = attend64(q[i, :, h].double(), k, v, seen, scale, coded(h) if coded else None)
            n = max(1, k.shape[0])
            bound = u * ref.abs() + mag * (u + 2 * (d + 8) * 2.0 ** -24 * size + (n + 64) * 2.0 ** -24) * (1 + u)
            if q.dtype == torch.float16:
                bound = bound + 2.0 ** -25 * (flat + 1)  # and the result's own subnormals
            bound = bound + 1e-37
            diff = (got[i, :, h].double() - ref).abs()
            assert torch.isfinite(diff).all(), (i, h)
            worst = max(worst, float((diff / bound).max())) if diff.numel() else worst
    assert worst <= 1.0, worst


def cross_case(dev, b, lq, lk, hq, hkv, d, dtype, seed, kb=None):
    g = seeded(seed)
    q, k, v = heads(g, dtype, b, lq, hq, d), heads(g, dtype, kb or b, lk, hkv, d), heads(g, dtype, kb or b, lk, hkv, d)
    return q.to(dev), k.to(dev), v.to(dev), g


def seen_of(b, lk, lengths, mask):
    seen = torch.ones(b, lk, dtype=torch.bool)
    if lengths is not None:
        seen &= torch.arange(lk) < torch.as_tensor(lengths)[:, None]
    if mask is not None:
        seen &= mask.cpu()
    return seen


def check_cross(got, q, k, v, seen, scale=None):
    b, lq, hq, d = q.shape
    per = hq // k.shape[2]

    def rows(i, h):
        at = i if k.shape[0] > 1 else 0
        keep = seen[i].to(q.device)
        kk, vv = (t[at, :, h // per][keep].double() for t in (k, v))
        return kk, vv, torch.ones(lq, kk.shape[0], dtype=torch.bool, device=q.device), scale or d ** -0.5

    check(got, q, rows)


# lengths around the tiles of 32 and 64 keys, rows around the blocks of 16, 32 and 128 (queries times heads of a K/V head)
CROSS = [
    (1, 1, 1, 1, 1, 64), (1, 1, 1, 4, 4, 128), (2, 1, 31, 8, 1, 128), (3, 1, 64, 12, 4, 64), (2, 1, 300, 32, 8, 128),
    (1, 3, 33, 7, 1, 128), (2, 5, 127, 14, 2, 64), (1, 32, 65, 2, 2, 128), (1, 33, 63, 1, 1, 64), (2, 16, 200, 4, 2, 128),
    (1, 17, 96, 2, 1, 128), (1, 127, 130, 2, 1, 128), (2, 130, 77, 3, 3, 64), (1, 300, 512, 2, 2, 128), (1, 1000, 40, 2, 1, 64),
    (1, 1, 5000, 2, 2, 128), (2, 4, 3001, 8, 2, 64), (40, 1, 129, 2, 1, 128), (1, 70, 2500, 4, 1, 128), (1, 129, 1900, 1, 1, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("b,lq,lk,hq,hkv,d", CROSS)
def test_cross_against_float64(dev, b, lq, lk, hq, hkv, d, dtype):
    from hy_nomas import attention

    q, k, v, g = cross_case(dev, b, lq, lk, hq, hkv, d, TYPES[dtype], b + lq * 3 + lk)
    lengths = torch.randint(0, lk + 1, (b,), generator=g)
    lengths[0] = lk
    if b > 1:
        lengths[1] = 0
    mask = torch.rand(b, lk, generator=g) < 0.6
    for what, n, m in (("none", None, None), ("lengths", lengths, None), ("mask", None, mask), ("both", lengths, mask)):
        print(f"cross b={b} lq={lq} lk={lk} hq={hq} hkv={hkv} d={d} {dtype} {what}", flush=True)
        got = attention.cross_attention(q, k, v, n.to(dev) if n is not None else None, m.to(dev) if m is not None else None)
        check_cross(got, q, k, v, seen_of(b, lk, n, m))


@pytest.mark.gpu
def test_cross_lengths_types_and_clamping(dev):
    from hy_nomas import attention

    q, k, v, _ = cross_case(dev, 4, 2, 100, 4, 2, 128, torch.bfloat16, 11)
    want = attention.cross_attention(q, k, v, torch.tensor([0, 100, 33, 100], device=dev))
    for n in (torch.tensor([-5, 1000, 33, 100], device=dev), torch.tensor([-2 ** 31, 2 ** 31 - 1, 33, 100], device=dev, dtype=torch.int32),
              torch.tensor([-2 ** 62, 2 ** 62, 33, 100], device=dev)):
        assert torch.equal(attention.cross_attention(q, k, v, n), want)
    assert (want[0] == 0).all()
    check_cross(want, q, k, v, seen_of(4, 100, [0, 100, 33, 100], None))
    strided = torch.tensor([[0, 9], [100, 9], [33, 9], [100, 9]], device=dev)[:, 0]
    assert torch.equal(attention.cross_attention(q, k, v, strided), want)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 40, 200])
@pytest.mark.parametrize("lk", [70, 1500])
def test_hidden_places_hold_anything(dev, lq, lk):
    """NaN and infinities at hidden keys and values, whole hidden tiles, hidden first and last keys: no trace of them."""
    from hy_nomas import attention

    q, k, v, g = cross_case(dev, 3, lq, lk, 4, 2, 128, torch.bfloat16, lq + lk)
    mask = (torch.rand(3, lk, generator=g) < 0.5).to(dev)
    mask[0, :66] = False
    mask[1, -65:] = False
    mask[2] = False
    want = attention.cross_attention(q, k, v, None, mask)
    check_cross(want, q, k, v, mask)
    assert (want[2] == 0).all()
    for bad in (float("nan"), float("inf"), -float("inf")):
        kb, vb = (torch.where(mask[:, :, None, None], t, torch.full_like(t, bad)) for t in (k, v))
        assert torch.equal(attention.cross_attention(q, kb, vb, None, mask), want)
    n = torch.tensor([lk - 3, 5, 0], device=dev)
    past = torch.arange(lk, device=dev) >= n[:, None]
    kb, vb = (t.masked_fill(past[:, :, None, None], float("nan")) for t in (k, v))
    assert torch.equal(attention.cross_attention(q, kb, vb, n), attention.cross_attention(q, k, v, n))


@pytest.mark.gpu
@pytest.mark.parametrize("lq,lk", [(1, 200), (60, 90), (3, 2000)])
def test_scores_of_every_size(dev, lq, lk):
    """Scores that leave all but one key no weight, that grow key by key, that are -inf or NaN at seen keys."""
    from hy_nomas import attention

    q, k, v, _ = cross_case(dev, 1, lq, lk, 2, 1, 128, torch.bfloat16, lk)
    ramp = torch.linspace(-40, 40, lk, device=dev)[None, :, None, None]
    for kk in (k * 30, (k * ramp).to(k.dtype), (k * ramp.flip(1)).to(k.dtype), torch.zeros_like(k)):
        got = attention.cross_attention(q, kk, v)
        check_cross(got, q, kk, v, seen_of(1, lk, None, None))
    dead = k.clone()
    dead[:, :70] = -float("inf")  # the first tiles score -inf for positive queries
    qp = q.abs()
    got = attention.cross_attention(qp, dead, v)
    check_cross(got, qp, dead[:, 70:], v[:, 70:], seen_of(1, lk - 70, None, None))
    dead[:] = -float("inf")
    assert (attention.cross_attention(qp, dead, v) == 0).all()
    dead = k.clone()
    dead[0, lk // 2, 0, 5] = float("nan")
    assert attention.cross_attention(q, dead, v).isnan().all()
    dead[0, lk // 2, 0, 5] = float("inf")  # a score of +inf has no softmax, as in the formula
    up = attention.cross_attention(qp, dead, v)
    assert up.isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [(1, 90), (150, 200)])
def test_layouts(dev, d, lq, lk):
    """Head-major operands, rows inside wider tensors, rows off a 16-byte boundary, one batch of states for all samples,
    overlapping views and an output of another layout give the contiguous call's bits."""
    from hy_nomas import attention

    q, k, v, g = cross_case(dev, 3, lq, lk, 4, 2, d, torch.bfloat16, d + lq, kb=1)
    n = torch.tensor([lk, 1, lk // 2], device=dev)
    mask = torch.rand(1, lk, generator=g).to(dev) < 0.7
    want = attention.cross_attention(q, k.expand(3, -1, -1, -1).contiguous(), v.expand(3, -1, -1, -1).contiguous(), n,
                                     mask.expand(3, -1).contiguous())
    check_cross(want, q, k, v, seen_of(3, lk, n.cpu(), mask.expand(3, -1)))

    def same(qq, kk, vv, nn=n, mm=mask, out=None):
        got = attention.cross_attention(qq, kk, vv, nn, mm, out=out)
        assert torch.equal(got, want) and (out is None or got is out)

    same(q, k, v)
    major = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    same(*major)
    for off in (8, 3):
        wide = [torch.zeros(*t.shape[:3], d + 16, device=dev, dtype=t.dtype) for t in (q, k, v)]
        for w, t in zip(wide, (q, k, v)):
            w[..., off:off + d] = t
        same(*(w[..., off:off + d] for w in wide))
    odd = torch.zeros(lk * 2 + 1, device=dev, dtype=torch.bool)
    odd[1::2] = mask[0]
    same(q, k, v, mm=odd[1::2][None])
    out = torch.full((3, 4, lq, d + 4), 7.0, device=dev, dtype=q.dtype)
    same(q, k, v, out=out[..., :d].transpose(1, 2))
    assert (out[..., d:] == 7).all()


def prefix_case(dev, b, lq, lp, ls, hq, hkv, d, dtype, int8, seed):
    from hy_nomas import kv

    g = seeded(seed)
    q, k, v = heads(g, dtype, b, lq, hq, d), heads(g, dtype, b, ls, hkv, d), heads(g, dtype, b, ls, hkv, d)
    pk, pv = heads(g, dtype, lp, hkv, d) * 1.5, heads(g, dtype, lp, hkv, d)
    prefix = tuple(tuple(x.to(dev) for x in kv.quantize_kv(t)) if int8 else t.to(dev) for t in (pk, pv))
    return q.to(dev), prefix, k.to(dev), v.to(dev), g


def check_prefix(got, q, prefix, k, v, lengths, causal, scale=None):
    b, lq, hq, d = q.shape
    per, ls = hq // k.shape[2], k.shape[1]
    coded = isinstance(prefix[0], tuple)
    pk, pv = (t[0].double() * t[1].double() if coded else t.double() for t in prefix)
    pk, pv = (t[0] if t.dim() == 4 else t for t in (pk, pv))

    def rows(i, h):
        n = ls if lengths is None else min(max(int(lengths[i]), 0), ls)
        kk, vv = (torch.cat([p[:, h // per], t[i if t.shape[0] > 1 else 0, :n, h // per].double()]) for p, t in ((pk, k), (pv, v)))
        lp = pk.shape[0]
        last = torch.full((lq, 1), lp + n, device=q.device)
        if causal:
            last = lp + (n - lq + 1 + torch.arange(lq, device=q.device)[:, None]).clamp(min=0)
        seen = torch.arange(lp + n, device=q.device) < last
        return kk, vv, seen, scale or d ** -0.5

    def codes(h):
        c, scales = (t[0] if t.dim() == 4 else t for t in prefix[1])
        return c[:, h // per], scales[:, h // per, 0]

    check(got, q, rows, codes if coded else None)


PREFIX = [
    # b, lq, lp, ls, hq, hkv, d
    (1, 1, 1, 0, 1, 1, 64), (1, 1, 64, 1, 4, 1, 128), (8, 1, 130, 20, 4, 1, 128), (8, 1, 2047, 129, 8, 2, 128),
    (3, 4, 33, 70, 6, 2, 64), (16, 4, 700, 60, 2, 2, 128), (64, 1, 500, 40, 8, 2, 128), (5, 7, 0, 100, 7, 1, 64),
    (2, 1, 0, 0, 2, 1, 128), (2, 33, 65, 33, 2, 2, 128), (4, 130, 300, 140, 2, 1, 64), (1, 200, 1000, 200, 2, 1, 128),
    (2, 300, 64, 310, 3, 1, 128), (1, 40, 5000, 40, 2, 2, 64), (33, 2, 4097, 3, 2, 2, 128), (2, 64, 1500, 900, 4, 2, 128),
]


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("b,lq,lp,ls,hq,hkv,d", PREFIX)
def test_prefix_against_float64(dev, b, lq, lp, ls, hq, hkv, d, int8):
    from hy_nomas import attention

    dtype = torch.float16 if (lq + lp) % 3 == 0 else torch.bfloat16
    q, prefix, k, v, g = prefix_case(dev, b, lq, lp, ls, hq, hkv, d, dtype, int8, lp + ls + b)
    lengths = torch.randint(0, ls + 1, (b,), generator=g)
    lengths[0] = ls
    for n in (None, lengths):
        for causal in (False, True):
            print(f"prefix b={b} lq={lq} lp={lp} ls={ls} hq={hq} hkv={hkv} d={d} {dtype} int8={int8} causal={causal} "
                  f"lengths={n is not None}", flush=True)
            got = attention.prefix_attention(q, prefix, k, v, n.to(dev) if n is not None else None, causal=causal)
            check_prefix(got, q, prefix, k, v, n, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 9, 40])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_value_scales_of_every_size(dev, dtype, lq):
    """Histories whose value scales span 2^-40 to 2^7 (the largest values stay in fp16): rows whose probability lies on keys of
    small values keep their precision beside keys of large ones, and a prefix of one size is as exact as its scale allows."""
    from hy_nomas import attention

    q, prefix, k, v, g = prefix_case(dev, 2, lq, 900, lq, 4, 2, 128, TYPES[dtype], True, 71 + lq)
    keys, (codes, scales) = prefix
    # the keys of value size i are those that queries of group i look at: a common direction, strongly
    group = torch.randint(0, 6, (900,), generator=g).to(dev)
    for h in range(2):
        for i in range(6):
            keys[0][group == i, h] = 0
            keys[0][group == i, h, 16 * i:16 * i + 16] = 100
    for j in range(lq):
        q[:, j] = 0.1 * q[:, j]
        q[:, j, :, 16 * (j % 6):16 * (j % 6) + 16] = 6.0
    keys[1].fill_(0.02)
    size = torch.tensor([2.0 ** -40, 2.0 ** -17, 2.0 ** -9, 0.02, 3.0, 128.0], device=dev)
    scales.copy_(size[group][:, None, None] * (1 + 0.5 * torch.rand(scales.shape, generator=g).to(dev)))
    for causal in (False, True):
        got = attention.prefix_attention(q, prefix, k, v, causal=causal)
        check_prefix(got, q, prefix, k, v, None, causal)
    for s in (0.0, 2.0 ** -60, 2.0 ** -24, 1.0, 400.0):  # (and 0: values of zero)
        scales.fill_(s)
        got = attention.prefix_attention(q, prefix, k, v)
        check_prefix(got, q, prefix, k, v, None, False)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_prefix_forms(dev, int8):
    """A leading batch of one, head-major and strided prefixes, a scale, an output and int32 lengths; own keys of one batch;
    dead rows of an own cache may hold NaN."""
    from hy_nomas import attention

    q, prefix, k, v, _ = prefix_case(dev, 3, 2, 150, 90, 4, 2, 128, torch.bfloat16, int8, 21)
    n = torch.tensor([90, 2, 41], device=dev)
    want = attention.prefix_attention(q, prefix, k, v, n, causal=True, scale=0.11)
    check_prefix(want, q, prefix, k, v, n, True, 0.11)

    def each(f):
        return tuple(tuple(f(x) for x in t) if isinstance(t, tuple) else f(t) for t in prefix)

    def wide(t):
        w = torch.zeros(t.shape[0], t.shape[1] + 3, t.shape[2] + 16, device=dev, dtype=t.dtype)
        w[:, 1:-2, : t.shape[2]] = t
        return w[:, 1:-2, : t.shape[2]]

    def off(t):
        w = torch.zeros(t.numel() + 1, device=dev, dtype=t.dtype)
        w[1:] = t.reshape(-1)
        return w[1:].view(t.shape)

    for p in (each(lambda t: t[None]), each(lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)), each(wide), each(off)):
        assert torch.equal(attention.prefix_attention(q, p, k, v, n.int(), causal=True, scale=0.11), want)
    past = torch.arange(90, device=dev) >= n[:, None]
    kb, vb = (t.masked_fill(past[:, :, None, None], float("nan")) for t in (k, v))
    out = torch.empty(2, 3, 4, 128, device=dev, dtype=q.dtype).transpose(0, 1)
    assert attention.prefix_attention(q, prefix, kb, vb, n, causal=True, scale=0.11, out=out) is out
    assert torch.equal(out, want)
    shared = attention.prefix_attention(q, prefix, k[:1], v[:1], n)
    check_prefix(shared, q, prefix, k[:1], v[:1], n, False)


@pytest.mark.gpu
def test_prefix_is_the_joined_attention(dev):
    """Samples that share a prefix answer as samples that each hold a copy of it."""
    from hy_nomas import attention

    q, prefix, k, v, _ = prefix_case(dev, 6, 1, 900, 50, 8, 4, 128, torch.bfloat16, False, 2)
    got = attention.prefix_attention(q, prefix, k, v)
    kk, vv = (torch.cat([p.expand(6, -1, -1, -1), t], 1) for p, t in zip(prefix, (k, v)))
    check_cross(got, q, kk, vv, seen_of(6, 950, None, None))
    check_cross(attention.cross_attention(q, kk, vv), q, kk, vv, seen_of(6, 950, None, None))


@pytest.mark.gpu
def test_offsets_past_32_bits(dev):
    """Keys whose element offsets from the tensor's start, and byte offsets from a sample's start, pass 2^31 and 2^32."""
    from hy_nomas import attention

    g = seeded(8)
    step = 1 << 22  # elements between keys: 600 keys are 2.5e9 elements, 5 GB
    store = torch.empty(600 * step + 4096, device=dev, dtype=torch.bfloat16)
    k, v = (torch.as_strided(store, (2, 300, 1, 128), (300 * step, step, 128, 1), at) for at in (0, 256))
    k.copy_(heads(g, k.dtype, *k.shape))
    v.copy_(heads(g, k.dtype, *v.shape))
    for lq in (1, 140):
        q = heads(g, k.dtype, 2, lq, 2, 128).to(dev)
        got = attention.cross_attention(q, k, v)
        check_cross(got, q, k.contiguous(), v.contiguous(), seen_of(2, 300, None, None))
        got = attention.prefix_attention(q, (k[1], v[1]), k[:, :70], v[:, :70])
        check_prefix(got, q, (k[1].contiguous(), v[1].contiguous()), k[:, :70].contiguous(), v[:, :70].contiguous(), None, False)


@pytest.mark.gpu
def test_token_strides_past_the_limit_are_copied(dev):
    from hy_nomas import attention

    step = (1 << 23) + 8
    store = torch.zeros(40 * step + 128, device=dev, dtype=torch.bfloat16)
    k = torch.as_strided(store, (1, 40, 1, 128), (0, step, 128, 1))
    k.copy_(heads(seeded(3), k.dtype, *k.shape))
    q = heads(seeded(4), k.dtype, 1, 3, 2, 128).to(dev)
    want = attention.cross_attention(q, k.contiguous(), k.contiguous())
    assert torch.equal(attention.cross_attention(q, k, k), want)
    assert torch.equal(attention.prefix_attention(q, (k[0], k[0]), k[:, :0], k[:, :0]), attention.prefix_attention(
        q, (k[0].contiguous(),) * 2, k[:, :0], k[:, :0]))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(12))
def test_seeded_shapes(dev, seed):
    """Shapes drawn over the kernels' row and key counts (few, half and whole blocks; one range of tiles and several)."""
    import random

    from hy_nomas import attention

    rng = random.Random(seed)
    hkv = rng.choice([1, 2, 3])
    hq, d, dtype = hkv * rng.choice([1, 2, 5]), rng.choice([64, 128]), rng.choice([torch.bfloat16, torch.float16])
    b, lq = rng.randint(1, 9), rng.choice([1, rng.randint(2, 12), rng.randint(13, 150)])
    lk, lp = rng.choice([rng.randint(1, 200), rng.randint(200, 6000)]), rng.choice([rng.randint(1, 300), rng.randint(300, 9000)])
    print(f"seed={seed} b={b} lq={lq} lk={lk} lp={lp} hq={hq} hkv={hkv} d={d} {dtype}", flush=True)
    q, k, v, g = cross_case(dev, b, lq, lk, hq, hkv, d, dtype, seed)
    n, mask = torch.randint(0, lk + 1, (b,), generator=g), torch.rand(b, lk, generator=g) < rng.random()
    check_cross(attention.cross_attention(q, k, v, n.to(dev), mask.to(dev)), q, k, v, seen_of(b, lk, n, mask))
    for int8 in (False, True):
        q, prefix, k, v, g = prefix_case(dev, b, lq, lp, lk, hq, hkv, d, dtype, int8, seed)
        for causal in (False, True):
            check_prefix(attention.prefix_attention(q, prefix, k, v, n.to(dev), causal=causal), q, prefix, k, v, n, causal)


@pytest.mark.gpu
def test_streams_repeats_and_replayed_graphs(dev):
    """The same bits on another stream, again and in a captured graph whose inputs, lengths and mask change between replays;
    two graphs of different sizes replayed in turn."""
    from hy_nomas import attention

    q, prefix, k, v, g = prefix_case(dev, 8, 1, 1500, 64, 8, 2, 128, torch.bfloat16, True, 5)
    n = torch.full((8,), 64, device=dev)
    ck, cv = k[:, :50].contiguous(), v[:, :50].contiguous()
    mask = torch.ones(8, 50, device=dev, dtype=torch.bool)

    def both():
        return attention.prefix_attention(q, prefix, k, v, n, causal=True), attention.cross_attention(q, ck, cv, n, mask)

    first = both()
    assert all(torch.equal(a, b) for a, b in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = both()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, second))
    graph, small = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    with torch.cuda.graph(small):
        other = attention.prefix_attention(q[:2], prefix, k[:2], v[:2], n[:2])
    for step in range(4):
        n.copy_(torch.randint(0, 65, (8,), generator=g))
        mask.copy_(torch.rand(8, 50, generator=g) < 0.5)
        q.copy_(heads(g, q.dtype, *q.shape))
        graph.replay()
        small.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, both()))
        assert torch.equal(other, attention.prefix_attention(q[:2], prefix, k[:2], v[:2], n[:2]))
        check_prefix(captured[0], q, prefix, k, v, n, True)


@pytest.mark.gpu
def test_calls_on_two_streams_at_once(dev):
    from hy_nomas import attention

    cases = [prefix_case(dev, 16, 1, 3000, 100, 8, 2, 128, torch.bfloat16, i == 1, i) for i in range(2)]
    want = [attention.prefix_attention(*c[:4]) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(10):
        for i, c in enumerate(cases):
            with torch.cuda.stream(streams[i]):
                got[i].append(attention.prefix_attention(*c[:4]))
    torch.cuda.synchronize()
    assert all(torch.equal(w, x) for w, xs in zip(want, got) for x in xs)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", ["fp8", "int8"])
def test_a_decoder_layer_serves_a_batch(dev, fmt):
    """One layer's step as a server runs it: quantizing norm, 8-bit linears, attention over the shared int8 prefix, cross
    attention to encoder states, the MLP's input norm; against the same steps with float64 norms and attentions.

    The streams are compared in norm.  A quantizer is off by half a code step at most: for e4m3 2^-4 of each value, evenly
    spread, so 2^-4 / sqrt(3) = 0.036 in norm, and independent from value to value, so a product of such values is that far
    off too; int8 in groups of 128, whose peak is four times their norm at most, 4 / 127 / sqrt(12) = 0.009.  Four quantizers
    lie before the last stream: 0.072 in quadrature if nothing else joined it; the last norm's codes add one: 0.081.  The
    roundings to bf16, 2^-9 each, are far below."""
    from hy_nomas import attention, kernels, kv

    b, hq, hkv, hd, dim, lp, ls, le = 6, 8, 2, 128, 1024, 700, 40, 90
    g = seeded(31)
    bf = torch.bfloat16

    def weight(n, k):
        w = torch.randn(n, k, generator=g) * k ** -0.5
        return kernels.quantize_activations(w.to(bf).to(dev), fmt, 128)

    x, r = torch.randn(b, dim, generator=g).to(bf).to(dev), torch.randn(b, dim, generator=g).to(bf).to(dev)
    w1, w2, w3 = ((1 + 0.1 * torch.randn(dim, generator=g)).to(bf).to(dev) for _ in range(3))
    wq, wo, wcq, wco = weight((hq + 2 * hkv) * hd, dim), weight(dim, hq * hd), weight(hq * hd, dim), weight(dim, hq * hd)
    prefix = tuple(kv.quantize_kv(heads(g, bf, lp, hkv, hd).to(dev)) for _ in range(2))
    ck, cv, ek, ev = (heads(g, bf, b, n, hkv, hd).to(dev) for n in (ls, ls, le, le))
    n = torch.tensor([1, 5, 40, 17, 33, 2], device=dev)
    en = torch.tensor([90, 0, 64, 65, 1, 33], device=dev)

    def layer(norm, linear, prefixed, crossed):
        k, v = ck.clone(), cv.clone()
        a, h = norm(x, r, w1)
        y = linear(a, wq).view(b, hq + 2 * hkv, hd)
        at = torch.arange(b, device=dev)
        k[at, n - 1], v[at, n - 1] = y[:, hq:hq + hkv].to(bf), y[:, hq + hkv:].to(bf)
        o = prefixed(y[:, None, :hq], k, v)
        a, h = norm(linear(o.reshape(b, -1), wo, True), h, w2)
        o = crossed(linear(a, wcq).view(b, 1, hq, hd))
        return norm(linear(o.reshape(b, -1), wco, True), h, w3)

    def norm(t, res, w):
        codes, scales, h = kernels.rms_norm_quant(t, w, res, kind=fmt, out=res if res is not r else None)
        return (codes, scales), h

    def linear(t, w, quantize=False):
        if quantize:
            return kernels.block_linear(t, *w, kind=fmt)
        return kernels.block_gemm(*t, *w, kind=fmt)

    (codes, scales), h = layer(norm, linear, lambda q, k, v: attention.prefix_attention(q, prefix, k, v, n, causal=True),
                               lambda q: attention.cross_attention(q, ek, ev, en))

    def norm64(t, res, w):
        s = t.double() + res.double()
        return s * torch.rsqrt(s.square().mean(-1, keepdim=True) + 1e-6) * w.double(), s

    def linear64(t, w, quantize=False):
        q, s = w
        return t.double() @ (q.float().double().view(q.shape[0], -1, 128) * s.double()[..., None]).view(q.shape[0], -1).t()

    def attend(q, keys):
        out = torch.zeros(b, 1, hq, hd, device=dev, dtype=torch.float64)
        for i in range(b):
            for j in range(hq):
                k, v = keys(i, j // (hq // hkv))
                if k.shape[0]:
                    out[i, 0, j] = torch.softmax(k @ q[i, 0, j].double() * hd ** -0.5, 0) @ v
        return out

    pk, pv = (t[0].double() * t[1].double() for t in prefix)
    ref, h64 = layer(norm64, linear64,
                     lambda q, k, v: attend(q, lambda i, j: (torch.cat([pk[:, j], k[i, :n[i], j].double()]), torch.cat([pv[:, j], v[i, :n[i], j].double()]))),
                     lambda q: attend(q, lambda i, j: (ek[i, :en[i], j].double(), ev[i, :en[i], j].double())))
    got = (codes.float().double().view(b, -1, 128) * scales.double()[..., None]).view(b, -1)
    for what, a, c, most in (("stream", h, h64, 0.072), ("norm", got, ref, 0.081)):
        off = float((a.double() - c).norm() / c.norm())
        assert off < most, (what, off)


def refused(name, match, *args, **kw):
    from hy_nomas import attention

    with pytest.raises(RuntimeError, match=match):
        getattr(attention, name)(*args, **kw)


def test_refusals_without_a_gpu(monkeypatch):
    from hy_nomas import _lib

    bf = torch.bfloat16

    def t(*shape, dtype=bf):
        return torch.zeros(*shape, dtype=dtype)

    q, k = t(2, 3, 4, 128), t(2, 5, 2, 128)
    p = (t(7, 2, 128), t(7, 2, 128))
    refused("cross_attention", "device tensors", q, k, k)
    refused("prefix_attention", "device tensors", q, p, k, k)
    monkeypatch.setattr(_lib, "require_device", lambda *t: None)
    for name, pre in (("cross_attention", ()), ("prefix_attention", (p,))):
        refused(name, "head dim 64 or 128", t(2, 3, 4, 96), *pre, t(2, 5, 2, 96), t(2, 5, 2, 96))
        refused(name, "bf16 or fp16", q.float(), *pre, k.float(), k.float())
        refused(name, "expected", q[0], *pre, k, k)
        refused(name, "do not match", q, *pre, k, t(2, 6, 2, 128))
        refused(name, "do not match", q, *pre, k.half(), k.half())
        refused(name, "do not match", q, *pre, t(2, 5, 3, 128), t(2, 5, 3, 128))
        refused(name, "do not match", q, *pre, t(2, 5, 0, 128), t(2, 5, 0, 128))
        refused(name, "do not match", q, *pre, t(3, 5, 2, 128), t(3, 5, 2, 128))
        refused(name, "lengths must be", q, *pre, k, k, torch.zeros(2))
        refused(name, "lengths must be", q, *pre, k, k, torch.zeros(3, dtype=torch.int32))
        refused(name, "out must be", q, *pre, k, k, out=t(2, 3, 4, 64))
        refused(name, "out must be", q, *pre, k, k, out=q.half())
        refused(name, "out must be", q, *pre, k, k, out=t(2, 3, 128, 4).transpose(2, 3))
        refused(name, "different devices", q, *pre, k, k.to("meta"))
        refused(name, "input's memory", q, *pre, k, k, out=q)
        refused(name, "input's memory", t(2, 5, 2, 128), *pre, k, k, out=k)
        refused(name, "expanded", q, *pre, k, k, out=t(1, 3, 4, 128).expand(2, 3, 4, 128))
        refused(name, "expanded", q, *pre, k, k, out=t(2, 1, 4, 128).expand(2, 3, 4, 128))
        for scale in (0.0, -1.0, 1e-31, float("nan"), float("inf")):
            refused(name, "scale", q, *pre, k, k, scale=scale)
    refused("cross_attention", "key_mask must be", q, k, k, None, t(2, 5))
    refused("cross_attention", "key_mask must be", q, k, k, None, torch.ones(2, 6, dtype=torch.bool))
    refused("prefix_attention", "prefix must be", q, p + p, k, k)
    refused("prefix_attention", "codes, scales", q, ((p[0].char(),), p[1]), k, k)
    shared = t(1, 6, 2, 128)
    for pre in ((shared, t(6, 2, 128)), (t(6, 2, 128), shared[0])):
        refused("prefix_attention", "input's memory", t(1, 6, 2, 128), pre, t(1, 5, 2, 128), t(1, 5, 2, 128), out=shared)
    refused("prefix_attention", "is not", q, (t(7, 3, 128), t(7, 3, 128)), k, k)
    refused("prefix_attention", "is not", q, (t(2, 7, 2, 128), t(2, 7, 2, 128)), k, k)
    refused("prefix_attention", "is not", q, (p[0].char(), p[1].char()), k, k)
    refused("prefix_attention", "differ", q, (p[0], t(8, 2, 128)), k, k)
    codes = (p[0].char(), torch.ones(7, 2, 1))
    refused("prefix_attention", "differ", q, (p[0], codes), k, k)
    refused("prefix_attention", "is not", q, ((p[0], codes[1]), codes), k, k)
    refused("prefix_attention", "do not match codes", q, ((codes[0], torch.ones(7, 2)), codes), k, k)
    refused("prefix_attention", "do not match codes", q, ((codes[0], codes[1].half()), codes), k, k)


def test_entry_point_refusals_without_a_gpu():
    from hy_nomas import _lib

    lib, p, big = _lib.lib(), 4096, 1 << 40  # never dereferenced: every call is refused on the host, or has no rows

    def cross(q=p, sq=(1536, 128, 512), k=p, sk=(1280, 128, 256), v=p, lengths=None, bits=0, mask=None, out=p, so=(1536, 128, 512), b=2,
              hq=4, hkv=2, lq=3, lk=5, d=128, dtype=0, scale=0.1, ws=p, nbytes=big):
        return lib.hn_cross_attention(q, *sq, k, *sk, v, *sk, lengths, bits, mask, 0, out, *so, b, hq, hkv, lq, lk, d, dtype, scale,
                                      ws, nbytes, None)

    bad = [dict(q=None), dict(out=None), dict(k=None), dict(v=None), dict(b=-1), dict(hq=0), dict(hkv=0), dict(hkv=3), dict(lq=-1),
           dict(lk=-1), dict(d=96), dict(dtype=2), dict(scale=0.0), dict(scale=float("nan")), dict(q=p + 8), dict(k=p + 2),
           dict(v=p + 4), dict(out=p + 4), dict(sq=(1536, 100, 512)), dict(sk=(1280, 128, 252)), dict(sk=(0, 0, 1 << 24)),
           dict(sk=(0, 0, -8)), dict(so=(1536, 130, 512)), dict(lengths=p, bits=16), dict(lengths=p + 4, bits=64),
           dict(lengths=p + 2, bits=32), dict(b=70000), dict(hq=70000, hkv=1), dict(lk=1 << 31), dict(lq=1 << 27)]
    for kw in bad:
        assert cross(**kw) == 1, kw
        assert b"hn_cross_attention" in lib.hn_last_error()
    assert cross(b=0) == 0 and cross(lq=0) == 0

    def prefix(table=(p, 128, 256, 0, 0, 0, p, 128, 256, 0, 0, 0), lp=7, ls=5, **kw):
        a = dict(q=p, k=p, v=p, out=p, b=2, hq=4, hkv=2, lq=3, d=128, dtype=0, scale=0.1, bits=0, lengths=None)
        a.update(kw)
        return lib.hn_prefix_attention(a["q"], 1536, 128, 512, _lib.int64s(table) if table else None, lp, a["k"], 1280, 128, 256, a["v"],
                                       1280, 128, 256, a["lengths"], a["bits"], 1, a["out"], 1536, 128, 512, a["b"], a["hq"], a["hkv"],
                                       a["lq"], ls, a["d"], a["dtype"], a["scale"], p, big, None)

    t = [p, 128, 256, 0, 0, 0, p, 128, 256, 0, 0, 0]
    for table in (None, [0] + t[1:], t[:6] + [0] + t[7:], [p + 2] + t[1:], t[:2] + [1 << 24] + t[3:], t[:3] + [p, 1, 2] + t[6:],
                  [p, 128, 264, p, 1, 2, p, 128, 256, p, 1, 2]):
        assert prefix(table) == 1, table
    for kw in (dict(lp=-1), dict(ls=-1), dict(hkv=3), dict(d=32), dict(k=None), dict(out=p + 4), dict(lengths=p, bits=8)):
        assert prefix(**kw) == 1, kw
        assert b"hn_prefix_attention" in lib.hn_last_error()
    assert prefix(b=0) == 0
    for f, n in ((lib.hn_cross_attention_workspace_bytes, 6), (lib.hn_prefix_attention_workspace_bytes, 7)):
        more = (0,) if n == 7 else ()
        assert f(*([1, 4, 2, 1, 10, 10, 128] if n == 7 else [1, 4, 2, 1, 10, 128]), *more) >= 0
        assert f(*([1, 4, 3, 1, 10, 10, 128] if n == 7 else [1, 4, 3, 1, 10, 128]), *more) == -1
        assert f(*([1, 4, 2, -1, 10, 10, 128] if n == 7 else [1, 4, 2, -1, 10, 128]), *more) == -1
        assert f(*([1, 4, 2, 1, 10, 10, 96] if n == 7 else [1, 4, 2, 1, 10, 96]), *more) == -1


def far_rows(dev, dtype, g, step, n, d, at=0):
    """[n, 1, d] values `step` elements apart in a store of their own."""
    t = torch.as_strided(torch.empty(n * step + at + d, device=dev, dtype=dtype), (n, 1, d), (step, d, 1), at)
    return t.copy_(heads(g, torch.float32, n, 1, d).to(dtype) if dtype.is_floating_point else
                   torch.randint(-127, 128, (n, 1, d), generator=g).to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("lq", [1, 40, 140])
@pytest.mark.parametrize("int8", [False, True])
def test_key_offsets_past_2_to_the_32(dev, lq, int8):
    """600 keys of one sample at the largest token stride, 2^23 elements: a tile's offset from the sample's start passes 2^32
    elements, 16-bit and int8 alike, and the scales' too, for few, half and whole blocks of rows."""
    from hy_nomas import attention

    g, step, n, d = seeded(lq), 1 << 23, 600, 128
    bf = torch.bfloat16
    q = heads(g, bf, 1, lq, 1, d).to(dev)
    if int8:
        prefix = tuple((far_rows(dev, torch.int8, g, step, n, d, 16 * i), far_rows(dev, torch.float32, g, step, n, 1).abs_().mul_(0.02))
                       for i in range(2))
        plain = tuple(tuple(t.contiguous() for t in p) for p in prefix)
    else:
        prefix = tuple(far_rows(dev, bf, g, step, n, d, 8 * i) for i in range(2))
        plain = tuple(t.contiguous() for t in prefix)
        got = attention.cross_attention(q, *(t[None] for t in prefix))
        check_cross(got, q, *(t[None] for t in plain), seen_of(1, n, None, None))
    k, v = (heads(g, bf, 1, 70, 1, d).to(dev) for _ in range(2))
    got = attention.prefix_attention(q, prefix, k, v)
    check_prefix(got, q, plain, k, v, None, False)


@pytest.mark.gpu
def test_an_output_whose_single_dims_have_odd_strides(dev):
    """A dimension of one element has no second row to misalign: its stride does not count."""
    from hy_nomas import attention

    g, bf = seeded(5), torch.bfloat16
    q, k, v = (heads(g, bf, 1, n, 2, 64).to(dev) for n in (3, 40, 40))
    out = torch.as_strided(torch.zeros(2 * 386, device=dev, dtype=bf), (1, 3, 2, 64), (386, 128, 64, 1))
    want = attention.cross_attention(q, k, v)
    assert attention.cross_attention(q, k, v, out=out) is out and torch.equal(out, want)
    out = torch.as_strided(torch.zeros(500, device=dev, dtype=bf), (1, 1, 2, 64), (7, 5, 64, 1))
    assert torch.equal(attention.cross_attention(q[:, :1], k, v, out=out), attention.cross_attention(q[:, :1], k, v))


# few, half and whole blocks of rows; one pass, two jobs and split keys; no prefix, a short, a long and an int8 one
LATER = [(2, 5, 0, 40, 2, 1, 128, False), (1, 12, 0, 3000, 4, 4, 64, False), (2, 20, 0, 90, 4, 2, 64, False), (2, 40, 0, 130, 2, 2, 128, False),
         (1, 150, 0, 200, 2, 1, 128, False), (2, 100, 33, 160, 4, 2, 64, False), (2, 130, 700, 140, 2, 1, 128, False), (4, 6, 900, 50, 4, 2, 128, False),
         (3, 9, 500, 70, 2, 2, 128, True), (2, 140, 300, 150, 2, 1, 64, True)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("b,lq,lp,ls,hq,hkv,d,int8", LATER)
def test_what_a_later_token_holds_stays_with_the_rows_that_see_it(dev, b, lq, lp, ls, hq, hkv, d, int8, dtype):
    """Under `causal`, infinities and NaN in keys and values from token j0 on: earlier queries' rows are those of the formula,
    later ones carry what they see, and a value's other dims stay as they are."""
    from hy_nomas import attention

    q, prefix, k, v, g = prefix_case(dev, b, lq, lp, ls, hq, hkv, d, TYPES[dtype], int8, lq + lp + 3)
    lengths = torch.full((b,), ls, device=dev)
    lengths[-1] = ls - 3
    clean = attention.prefix_attention(q, prefix, k, v, lengths, causal=True)
    check_prefix(clean, q, prefix, k, v, lengths, True)
    for j0 in sorted({1, lq // 2, lq - 1}):
        for what, bad in (("values", "nan"), ("values", "inf"), ("keys", "nan"), ("keys", "inf"), ("both", "-inf")):
            print(f"later b={b} lq={lq} lp={lp} ls={ls} d={d} int8={int8} {dtype} j0={j0} {what} {bad}", flush=True)
            kb, vb = k.clone(), v.clone()
            for i in range(b):
                n = int(lengths[i])
                if what != "values":
                    kb[i, n - lq + j0:n] = float(bad)
                if what != "keys":
                    vb[i, n - lq + j0:n, :, 5] = float(bad)
                if what == "both":
                    vb[i, n - lq + j0:n] = float(bad)
            got = attention.prefix_attention(q, prefix, kb, vb, lengths, causal=True)
            check_prefix(got[:, :j0], q[:, :j0], prefix, k, v, lengths - (lq - j0), True)
            if what == "values":
                assert not got[:, j0:, :, 5].isfinite().any()
                rest = got.clone()
                rest[..., 5] = clean[..., 5]
                check_prefix(rest, q, prefix, k, v, lengths, True)
            elif bad == "nan":
                assert got[:, j0:].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("b,lq,ls,hq,hkv,d", [(2, 150, 140, 2, 2, 64), (2, 12, 10, 2, 1, 128), (2, 40, 30, 2, 2, 128), (1, 300, 260, 2, 1, 128)])
def test_queries_before_the_first_own_key_give_zeros_beside_anything(dev, b, lq, ls, hq, hkv, d):
    """More queries than own keys and no prefix: the first queries see nothing, whatever the keys of the others hold."""
    from hy_nomas import attention

    q, prefix, k, v, _ = prefix_case(dev, b, lq, 0, ls, hq, hkv, d, torch.bfloat16, False, lq)
    for what in (k, v):
        what[:] = float("nan")
        got = attention.prefix_attention(q, prefix, k, v, causal=True)
        assert (got[:, :lq - ls] == 0).all() and got[:, lq - ls:].isnan().all()
        what[:] = 1.0
