"""Grouped-head attention at the ends of the numbers' range, in every kernel: scores far past 2^24, whose fp32 spacing is
more than one, and values whose sums come near fp32's largest."""

from __future__ import annotations

import pytest
import torch

from minisgl_amd.kernel import lib
from test_gqa_gpu import DEV, InBlocks, Paged, i32, padding, prompt_in_blocks, run_prompt

pytestmark = pytest.mark.gpu
NAN = float("nan")


class Exact:
    """Attention of one request in 64 bits: ``q [E, Hq, D]`` over ``k, v [L, Hkv, D]``, head by head."""

    def __init__(self, q, k, v, scale):
        E, Hq, _ = q.shape
        L, Hkv, _ = k.shape
        seen = (torch.arange(L) <= (L - E + torch.arange(E))[:, None]).to(DEV)
        out, top, lse, size = [], [], [], []
        for h in range(Hq):
            kh, vh = k[:, h * Hkv // Hq].to(DEV).double(), v[:, h * Hkv // Hq].to(DEV).double()
            s = torch.where(seen, q[:, h].to(DEV).double() @ kh.t() * scale, -float("inf"))
            top.append(s.amax(-1)), lse.append(torch.logsumexp(s, -1))
            p = torch.exp(s - lse[-1][:, None])
            out.append(p @ vh), size.append(p @ vh.abs())
        self.out, self.size = torch.stack(out, 1), torch.stack(size, 1)
        self.top, self.lse, self.keys = torch.stack(top, 1), torch.stack(lse, 1), L

    def check(self, out, lse, what=""):
        """For scores that are one exact product each: the kernels round the scaled score (and their constant scale times
        log2 e), 2^-22 of it at most. That moves a weight by as much while |top| is below 2^13; from there on the nearest
        other bf16 key is 2^-8 |top| >= 32 away and weighs nothing, and keys that are alike have rounded alike. Numerators
        and results are rounded to bf16, half a step each; sums have L roundings."""
        out, lse = out.to(DEV).double(), lse.to(DEV).double()
        moved = (2.0 ** -22 * (self.top.abs() + 200)).clamp_max(2.0 ** -9)
        rel = 2.0 ** -8 + 2 * moved + 2 * (self.keys + 16) * 2.0 ** -24
        bound = 1.02 * (rel[..., None] * self.size + 2.0 ** -8 * self.out.abs())
        assert out.isfinite().all() and lse.isfinite().all(), what
        over = (out - self.out).abs() - bound
        assert over.max() <= 0, f"{what}: out is {float(over.max()):.3e} past its bound"
        off = (lse - self.lse).abs() - (2.0 ** -21 * (self.lse.abs() + 200) + (self.keys + 16) * 2.0 ** -24)
        assert off.max() <= 0, f"{what}: lse is {float(off.max()):.3e} past its bound"


def far(gen, tokens, q_heads, keys, kv_heads, dim, rising=False):
    """Queries and keys of one dimension: scores of exact products, from hundreds to 2^34, of either sign."""
    q, k = torch.zeros((tokens, q_heads, dim)), torch.zeros((keys, kv_heads, dim))
    at = int(torch.randint(0, dim, (1,), generator=gen))
    sign = torch.randint(0, 2, (tokens, q_heads), generator=gen) * 2.0 - 1
    q[..., at] = sign * 2.0 ** torch.randint(0, 22, (tokens, q_heads), generator=gen)
    k[..., at] = torch.randn((keys, kv_heads), generator=gen) * 4096
    if rising:
        k[..., at] = (torch.arange(keys)[:, None] - keys / 3) * 16
    return q.to(torch.bfloat16), k.to(torch.bfloat16)


@pytest.mark.parametrize("rising", [False, True])
@pytest.mark.parametrize("lens,heads,dim,blocks", [
    ([300, 1, 77], (8, 2), 128, False), ([300, 1, 77], (8, 2), 64, False),  # 16-row CTAs
    ([300, 1, 77], (8, 2), 128, True), ([700, 33], (6, 2), 64, True),  # blocks of 128 rows
    ([2100], (6, 2), 64, False), ([4100], (4, 1), 128, False),  # in two halves of the keys
    ([2600], (51, 17), 128, False),  # blocks of 256 rows
])
def test_far_scores_of_prompts(lens, heads, dim, blocks, rising):
    gen = torch.Generator().manual_seed(sum(lens))
    q, k = far(gen, sum(lens), heads[0], sum(lens), heads[1], dim, rising)
    v = torch.randn((sum(lens), heads[1], dim), generator=gen).to(torch.bfloat16)
    out, lse = (prompt_in_blocks if blocks else run_prompt)(q, k, v, lens, 0.125)
    at = 0
    for n in lens:
        one = slice(at, at + n)
        Exact(q[one], k[one], v[one], 0.125).check(out[one], lse[one], f"{n} of {lens}")
        at += n


@pytest.mark.parametrize("kind,extends,prefixes,heads", [
    (Paged, [1, 1], [3000, 40], (8, 2)), (Paged, [3, 2], [5000, 600], (16, 4)),  # streamed, split and joined
    (InBlocks, [200, 3], [3000, 700], (8, 2)), (InBlocks, [90, 40], [300, 64], (6, 2)),  # blocks, split and in one piece
])
@pytest.mark.parametrize("dim", [64, 128])
def test_far_scores_over_pages(kind, extends, prefixes, heads, dim):
    """Keys split over pieces: each piece's largest score is its own, and one key of the prefix wins for either sign."""
    gen = torch.Generator().manual_seed(dim + len(extends))
    c = kind(extends, prefixes, *heads, dim, 16, seed=dim, scale=0.125)
    rows, keys, at = [], [], 0
    for b, (e, n) in enumerate(zip(extends, c.lens)):
        q, k = far(gen, e, heads[0], n, heads[1], dim)
        one = k.abs().amax((0, 1)).argmax()
        k[..., one] *= 0.25
        k[prefixes[b] // 3, :, one], k[prefixes[b] // 2, :, one] = 24576.0, -24576.0
        j = torch.arange(n)
        rows.append(c.pt[b].long()[j // 16] * 16 + j % 16)
        c.k.view(-1, heads[1], dim)[rows[-1]] = k
        c.q[at : at + e] = q
        keys.append(k)
        at += e
    out, lse = c.run()
    at = 0
    for e, k, r in zip(extends, keys, rows):
        one = slice(at, at + e)
        Exact(c.q[one], k, c.v.view(-1, heads[1], dim)[r], 0.125).check(out[one], lse[one])
        at += e


@pytest.mark.parametrize("blocks", [False, True])
def test_far_scores_beside_a_later_token_that_is_not_finite(blocks):
    """A row computed again by itself, its scores summed in another order than the product's."""
    gen = torch.Generator().manual_seed(9)
    n, hq, hk, dim = 150, 4, 2, 128
    q, k = far(gen, n, hq, n, hk, dim)
    v = torch.randn((n, hk, dim), generator=gen).to(torch.bfloat16)
    want = Exact(q[:-1], k[:-1], v[:-1], 0.125)
    v[-1] = NAN
    out, lse = (prompt_in_blocks if blocks else run_prompt)(q, k, v, [n], 0.125)
    want.check(out[:-1], lse[:-1])
    assert not out[-1].isfinite().any()


@pytest.mark.parametrize("extends", [[1, 2], [140]])
@pytest.mark.parametrize("blocks", [False, True])
def test_far_scores_of_full_rows(extends, blocks):
    """Scores of about 1e10 that are sums over all dimensions: their fp32 sums differ by more than one, so a row's weights
    are only known to be some average of its values; no sum may pass for no keys, or leave the range."""
    c = (InBlocks if blocks else Paged)(extends, [300] * len(extends), 8, 2, 128, 16, seed=5, scale=1e10 * 128 ** -0.5)
    c.v = c.v.abs() + 0.5
    out, lse = c.run()
    ref = c.ref()
    assert out.isfinite().all() and lse.isfinite().all() and float(out.float().min()) >= 0.49
    assert ((lse.double().cpu() - ref.lse).abs() <= ref.lse_bound).all()


def rising_scores(gen, tokens, q_heads, keys, kv_heads, dim, nats):
    """Queries and keys of one dimension, scores (at scale 0.125) rising by ``nats`` over the keys."""
    q, k = torch.zeros((tokens, q_heads, dim)), torch.zeros((keys, kv_heads, dim))
    at = int(torch.randint(0, dim, (1,), generator=gen))
    q[..., at] = 8.0
    k[..., at] = torch.linspace(-nats / 2, nats / 2, keys)[:, None]
    return q.to(torch.bfloat16), k.to(torch.bfloat16)


def huge(gen, *shape, most):
    """Values of either sign, from 1 to 2^most."""
    size = 2.0 ** (torch.rand(shape, generator=gen) * most)
    return (size * (torch.randint(0, 2, shape, generator=gen) * 2 - 1)).to(torch.bfloat16)


PROMPTS = [([300, 1, 77], (8, 2), 128, False), ([300, 1, 77], (8, 2), 64, False), ([300, 1, 77], (8, 2), 128, True),
           ([700, 33], (6, 2), 64, True), ([2100], (6, 2), 64, False), ([4100], (4, 1), 128, False), ([2600], (51, 17), 128, False)]


@pytest.mark.parametrize("lens,heads,dim,blocks", PROMPTS)
def test_values_near_the_largest_of_prompts(lens, heads, dim, blocks):
    """Finite values whose weighted sums are finite, under scores whose largest comes last: no partial sum may pass
    fp32's range for good."""
    gen = torch.Generator().manual_seed(sum(lens))
    for nats, most in ((20, 100), (60, 126)):
        if most == 126 and max(lens) > 1000:
            continue  # every row is computed again by itself
        q, k, v = [], [], []
        for n in lens:
            for x, y in zip((q, k), rising_scores(gen, n, heads[0], n, heads[1], dim, nats)):
                x.append(y)
            v.append(huge(gen, n, heads[1], dim, most=most))
        out, lse = (prompt_in_blocks if blocks else run_prompt)(torch.cat(q), torch.cat(k), torch.cat(v), lens, 0.125)
        at = 0
        for n, x, y, z in zip(lens, q, k, v):
            one = slice(at, at + n)
            Exact(x, y, z, 0.125).check(out[one], lse[one], f"{n} of {lens}, {nats} nats, up to 2^{most}")
            at += n


@pytest.mark.parametrize("kind,extends,prefixes,heads", [
    (Paged, [1, 1], [3000, 40], (8, 2)), (Paged, [3, 2], [5000, 600], (16, 4)), (Paged, [20], [300], (8, 2)),
    (InBlocks, [200, 3], [3000, 700], (8, 2)), (InBlocks, [90, 40], [300, 64], (6, 2)),
])
@pytest.mark.parametrize("dim", [64, 128])
def test_values_near_the_largest_over_pages(kind, extends, prefixes, heads, dim):
    """Keys of low scores and values near the largest before keys of high scores and ordinary values, which are the
    result; and a rise over all keys."""
    gen = torch.Generator().manual_seed(dim + len(extends))
    for low in (False, True):
        c = kind(extends, prefixes, *heads, dim, 16, seed=dim, scale=0.125)
        made, at = [], 0
        for b, (e, n) in enumerate(zip(extends, c.lens)):
            q, k = rising_scores(gen, e, heads[0], n, heads[1], dim, 60)
            v = huge(gen, n, heads[1], dim, most=100)
            if low:
                half = prefixes[b] * 2 // 3
                k[:half] = -k[:half].abs() - (k != 0)[:half] * 200.0
                v[:half], v[half:] = 2.0 ** 127, torch.randn(v[half:].shape, generator=gen).to(torch.bfloat16)
            j = torch.arange(n)
            rows = c.pt[b].long()[j // 16] * 16 + j % 16
            c.k.view(-1, heads[1], dim)[rows], c.v.view(-1, heads[1], dim)[rows] = k, v
            c.q[at : at + e] = q
            made.append((slice(at, at + e), q, k, v))
            at += e
        out, lse = c.run()
        for one, q, k, v in made:
            Exact(q, k, v, 0.125).check(out[one], lse[one], f"low {low}")


@pytest.mark.parametrize("lens,heads,dim,blocks", PROMPTS[:6])
def test_an_infinity_that_rows_attend_stays_what_it_is(lens, heads, dim, blocks):
    """One dimension of one token is infinite: the rows from it on are so in that dimension alone, beside a later token
    that is NaN too; a token of both signs' infinity gives NaN."""
    gen = torch.Generator().manual_seed(dim)
    randn = lambda h: torch.randn((sum(lens), h, dim), generator=gen).to(torch.bfloat16)  # noqa: E731
    q, k, v = randn(heads[0]), randn(heads[1]), randn(heads[1])
    n, x = lens[0], lens[0] // 3
    want = Exact(q[:n], k[:n], v[:n], 0.125)
    for later in (False, True):
        w = v.clone()
        w[x, :, 5], w[x + 7, :, 9], w[x + 8, :, 9] = -float("inf"), float("inf"), -float("inf")
        if later:
            w[n - 1] = NAN
        out, lse = (prompt_in_blocks if blocks else run_prompt)(q, k, w, lens, 0.125)
        out, lse, rows = out[:n], lse[:n], n - later
        assert (out[x:rows, :, 5] == -float("inf")).all() and out[x + 8 : rows, :, 9].isnan().all() and (out[x + 7, :, 9] == float("inf")).all()
        assert not later or out[n - 1].isnan().all()
        fixed = out.clone()
        fixed[x:, :, 5], fixed[x + 7 :, :, 9] = want.out[x:, :, 5].to(out), want.out[x + 7 :, :, 9].to(out)
        if later:
            fixed[n - 1] = want.out[n - 1].to(out)
        want.check(fixed, lse)


@pytest.mark.parametrize("n,heads,tokens,most", [(300, (8, 1), 1, 1 << 17), (64, (8, 2), 1, 1 << 19), (300, (8, 1), 3, 1 << 17), (40, (8, 1), 20, 1 << 20)])
def test_split_keys_whose_sum_passes_24_bits(n, heads, tokens, most):
    """Long requests on one shared prefix: the lengths' sum, by which both kernels of the call find the pieces, is past
    what fp32 counts one by one. More requests than a wave has lanes, and few."""
    gen = torch.Generator().manual_seed(n + tokens)
    dim, ps, (hq, hk) = 64, 64, heads
    on_gpu = torch.Generator(device=DEV).manual_seed(n)
    k, v = (torch.randn((most // ps, ps, hk, dim), generator=on_gpu, device=DEV, dtype=torch.bfloat16) for _ in range(2))
    pt = torch.randperm(most // ps, generator=gen).to(torch.int32)
    lens = torch.randint(most // 4, most + 1, (n,), generator=gen).tolist()
    lens[:3] = [most, tokens, most - 1]
    assert sum(lens) > 1 << 24
    q = torch.randn((n * tokens, hq, dim), generator=gen).to(torch.bfloat16).to(DEV)
    out, lse = torch.full_like(q, NAN), torch.full((n * tokens, hq), NAN, device=DEV)
    lib.gqa_chunk(q, k, v, pt.to(DEV).expand(n, -1).contiguous(), i32(list(range(0, n * tokens + 1, tokens))), i32(lens), tokens, 0.125, out, lse)
    torch.cuda.synchronize()
    rows = (pt.long()[:, None] * ps + torch.arange(ps)).flatten().to(DEV)
    over = []
    for h in range(hk):
        k64, v64 = (x.view(-1, hk, dim)[rows, h].double() for x in (k, v))
        size64 = v64.abs()
        group = slice(h * hq // hk, (h + 1) * hq // hk)
        for b, L in enumerate(lens):
            one = slice(b * tokens, (b + 1) * tokens)
            s = torch.matmul(k64[:L], q[one, group].double().flatten(0, 1).t().contiguous()).t().reshape(tokens, -1, L) * 0.125
            for i in range(tokens - 1):
                s[i, :, L - tokens + 1 + i :] = -float("inf")
            z = torch.logsumexp(s, -1)
            p = torch.exp(s - z[..., None]).flatten(0, 1)
            cut = -(-L // 4096)
            p = torch.nn.functional.pad(p, (0, cut * 4096 - L)).view(-1, cut, 4096).transpose(0, 1).contiguous()
            ref, size = (torch.bmm(p, x[: cut * 4096].view(cut, 4096, dim)).sum(0).view(tokens, -1, dim) for x in (v64, size64))
            # scores are sums of D products, sum |q k| scale <= 200 here: (D + 16) roundings of 2^-24
            delta = (dim + 16) * 2.0 ** -24 * 200
            rel = 2.0 ** -8 + 2 * delta + 2 * (L + 16) * 2.0 ** -24
            over.append(((out[one, group].double() - ref).abs() - 1.02 * (rel * size + 2.0 ** -8 * ref.abs())).max())
            over.append(((lse[one, group].double() - z).abs() - (delta + (L + 16) * 2.0 ** -24 + 2.0 ** -22 * z.abs())).max())
    assert float(torch.stack(over).max()) <= 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [NAN, float("inf"), -float("inf")])
@pytest.mark.parametrize("blocks", [False, True])
def test_every_head_of_a_token_whose_key_is_not_finite(dim, value, blocks):
    """Queries of both signs make such a score NaN: no head and no dimension of the rows that attend it is finite, and
    the rows before are as they were."""
    gen = torch.Generator().manual_seed(31)
    lens, last = [200, 70], [198, 199, 269]
    q, k, v = (torch.randn((270, h, dim), generator=gen).to(torch.bfloat16) for h in (6, 2, 2))
    call = prompt_in_blocks if blocks else run_prompt
    clean, clean_lse = call(q, k, v, lens, 0.1)
    for t in (k, v):
        t[last] = value
    out, lse = call(q, k, v, lens, 0.1)
    assert not out[last].isfinite().any() and not lse[last].isfinite().any()
    keep = [i for i in range(270) if i not in last]
    assert out[keep].isfinite().all() and torch.equal(lse[keep], clean_lse[keep])
    # computed again in fp32 or as before: numerators rounded to bf16 or not, results rounded twice
    assert ((out[keep].double() - clean[keep].double()).abs() <= 2.0 ** -7 * 4 + 2.0 ** -7 * clean[keep].double().abs()).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[2999, 4] * 32, [20000, 3] * 32, [30000] + [2100] * 40, [17000, 300, 1] * 20, [5000] * 40 + [64] * 24])
def test_pieces_enlarged_until_they_run_at_once(dim, lens):
    """At most 64 requests of few CTAs, cut into more pieces at first than run at once (512 of two KV heads)."""
    first = max((2 * sum((n + 15) // 16 * 16 for n in lens) // 512 + 64) // 64 * 64, 128)  # keys of a piece
    assert 2 * sum(-(-n // first) for n in lens) > 512
    c = Paged([1] * len(lens), [n - 1 for n in lens], 8, 2, dim, 16, seed=len(lens))
    for out, lse in (c.decode(), c.run()):
        at = 0
        for b, n in enumerate(lens):
            rows = c.pt[b].long()[torch.arange(n) // 16] * 16 + torch.arange(n) % 16
            ref = Exact(c.q[b : b + 1], c.k.view(-1, 2, dim)[rows], c.v.view(-1, 2, dim)[rows], c.scale)
            rel = 2.0 ** -8 + 2 * (dim + 16) * 2.0 ** -24 * 200 + 2 * (n + 16) * 2.0 ** -24
            assert ((out[b : b + 1].double() - ref.out).abs() <= 1.02 * (rel * ref.size + 2.0 ** -8 * ref.out.abs())).all(), (b, n)
            assert ((lse[b : b + 1].double() - ref.lse).abs() <= (dim + 16) * 2.0 ** -24 * 200 + (n + 16) * 2.0 ** -24 + 2.0 ** -22 * ref.lse.abs()).all(), (b, n)


@pytest.mark.parametrize("kind,extends,prefixes,heads", [
    (Paged, [1, 1, 1], [3000, 40, 1999], (8, 2)), (Paged, [3, 2], [5000, 1111], (16, 4)), (InBlocks, [200, 3], [3000, 700], (8, 2)),
])
@pytest.mark.parametrize("dim", [64, 128])
def test_keys_alike_at_far_scores_weigh_alike_in_every_piece(kind, extends, prefixes, heads, dim):
    """All scores of a row are one number, in most rows past what fp32 adds a sum's logarithm to: the result is the mean
    of all values, however many keys a piece of them holds."""
    gen = torch.Generator().manual_seed(dim)
    c = kind(extends, prefixes, *heads, dim, 16, seed=dim + 1, scale=0.125)
    made, at = [], 0
    for b, (e, n) in enumerate(zip(extends, c.lens)):
        q, k = far(gen, e, heads[0], n, heads[1], dim)
        k[:] = (k != 0) * 1536.0 if b % 2 else (k != 0) * -640.0
        v = torch.randn((n, heads[1], dim), generator=gen) + torch.arange(n)[:, None, None] * (4.0 / n)  # pieces differ
        j = torch.arange(n)
        rows = c.pt[b].long()[j // 16] * 16 + j % 16
        c.k.view(-1, heads[1], dim)[rows], c.v.view(-1, heads[1], dim)[rows] = k.to(torch.bfloat16), v.to(torch.bfloat16)
        c.q[at : at + e] = q
        made.append((slice(at, at + e), q, k.to(torch.bfloat16), v.to(torch.bfloat16)))
        at += e
    out, lse = c.run()
    for one, q, k, v in made:
        Exact(q, k, v, 0.125).check(out[one], lse[one])
