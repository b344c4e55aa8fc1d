"""Grouped-head attention on the GPU (packed prompts, chunks and single tokens over a paged cache) against the 64-bit
oracle, within the bounds that oracle/ref_gqa.py derives from the kernels' roundings."""

from __future__ import annotations

import random

import pytest
import torch

from minisgl_amd.kernel import lib
from oracle import ref_gqa as R

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
NAN = float("nan")


def randn(gen, *shape):
    return torch.randn(shape, generator=gen).to(torch.bfloat16)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def cumulative(x):
    out = [0]
    for v in x:
        out.append(out[-1] + v)
    return out


def check(out, lse, ref, what=""):
    out, lse = out.double().cpu(), lse.double().cpu()
    same = lambda a, b: torch.equal(torch.isinf(a), torch.isinf(b))  # noqa: E731
    assert not out.isnan().any() and not lse.isnan().any() and same(lse, ref.lse), what
    over = (out - ref.out).abs() - ref.out_bound
    assert over.max() <= 0, f"{what}: out is {over.max():.3e} past its bound"
    off = torch.where(ref.lse.isinf(), 0.0, lse - ref.lse).abs() - ref.lse_bound
    assert off.max() <= 0, f"{what}: lse is {off.max():.3e} past its bound"


class Paged:
    """A batch over a pool with NaN in every row that no request owns, and past every length."""

    def __init__(self, extends, prefixes, q_heads, kv_heads, dim, page_size, seed, spare_rows=0, scale=None):
        gen = torch.Generator().manual_seed(seed)
        self.extends, self.lens = list(extends), [e + p for e, p in zip(extends, prefixes)]
        self.scale = dim ** -0.5 if scale is None else scale
        need = [-(-n // page_size) for n in self.lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen).to(torch.int32)
        self.k = torch.full((pages, page_size, kv_heads, dim), NAN, dtype=torch.bfloat16)
        self.v = torch.full_like(self.k, NAN)
        self.pt = torch.full((len(need), max(max(need), 1)), -7, dtype=torch.int32)  # unused entries are no pages
        at = 0
        for b, (n, L) in enumerate(zip(need, self.lens)):
            self.pt[b, :n] = order[at : at + n]
            at += n
            j = torch.arange(L)
            rows = self.pt[b].long()[j // page_size] * page_size + j % page_size
            self.k.view(-1, kv_heads, dim)[rows] = randn(gen, L, kv_heads, dim)
            self.v.view(-1, kv_heads, dim)[rows] = randn(gen, L, kv_heads, dim)
        self.T = sum(self.extends)
        self.q = randn(gen, self.T + spare_rows, q_heads, dim)

    def ref(self):
        return R.chunk(self.q, self.k, self.v, self.pt, self.extends, self.lens, self.scale)

    def run(self, max_q=None, workspace=None):
        q = self.q.to(DEV)
        out = torch.full_like(q, NAN)
        lse = torch.full(q.shape[:2], NAN, device=DEV)
        lib.gqa_chunk(q, self.k.to(DEV), self.v.to(DEV), self.pt.to(DEV), i32(cumulative(self.extends)), i32(self.lens),
                      max(self.extends) if max_q is None else max_q, self.scale, out, lse, workspace)
        torch.cuda.synchronize()
        return out, lse

    def decode(self):
        q = self.q.to(DEV)
        out = torch.full_like(q, NAN)
        lse = torch.full(q.shape[:2], NAN, device=DEV)
        lib.gqa_decode(q, self.k.to(DEV), self.v.to(DEV), self.pt.to(DEV), i32(self.lens), self.scale, out, lse)
        torch.cuda.synchronize()
        return out, lse


def run_prompt(q, k, v, lens, scale):
    out = torch.full(q.shape, NAN, dtype=torch.bfloat16, device=DEV)
    lse = torch.full(q.shape[:2], NAN, device=DEV)
    lib.gqa_prompt(q.to(DEV), k.to(DEV), v.to(DEV), i32(cumulative(lens)), scale, out, lse)
    torch.cuda.synchronize()
    return out, lse


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (4, 4), (6, 2), (14, 2), (20, 4), (48, 3)])
def test_prompt_heads(dim, heads):
    gen = torch.Generator().manual_seed(heads[0] * dim)
    lens = [33, 1, 0, 129, 64]
    q, k, v = randn(gen, sum(lens), heads[0], dim), randn(gen, sum(lens), heads[1], dim), randn(gen, sum(lens), heads[1], dim)
    out, lse = run_prompt(q, k, v, lens, dim ** -0.5)
    check(out, lse, R.prompt(q, k, v, lens, dim ** -0.5))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [127, 128, 129], [255, 257], [1500, 3, 700], [2049]])
def test_prompt_lengths(dim, lens):
    gen = torch.Generator().manual_seed(sum(lens))
    q, k, v = randn(gen, sum(lens), 4, dim), randn(gen, sum(lens), 2, dim), randn(gen, sum(lens), 2, dim)
    out, lse = run_prompt(q, k, v, lens, dim ** -0.5)
    check(out, lse, R.prompt(q, k, v, lens, dim ** -0.5))


def test_prompt_many_requests():
    """More requests than a wave has lanes, empty ones among them."""
    r = random.Random(5)
    lens = [r.choice([0, 1, 2, 17, 40]) for _ in range(150)]
    gen = torch.Generator().manual_seed(5)
    q, k, v = randn(gen, sum(lens), 6, 64), randn(gen, sum(lens), 3, 64), randn(gen, sum(lens), 3, 64)
    out, lse = run_prompt(q, k, v, lens, 0.2)
    check(out, lse, R.prompt(q, k, v, lens, 0.2))


def test_prompt_strided():
    """q, k and v as views of one projection output, out and lse with strides of their own (out heads first), rows behind
    the last sequence untouched."""
    gen = torch.Generator().manual_seed(3)
    lens, hq, hk, d, spare = [70, 201], 8, 2, 128, 9
    T = sum(lens)
    qkv = randn(gen, T + spare, (hq + 2 * hk) * d + 8)
    dev = qkv.to(DEV)
    views = lambda x: (x[:, : hq * d].unflatten(1, (hq, d)), x[:, hq * d : (hq + hk) * d].unflatten(1, (hk, d)),  # noqa: E731
                       x[:, (hq + hk) * d : (hq + 2 * hk) * d].unflatten(1, (hk, d)))
    q, k, v = views(dev)
    ref = R.prompt(*views(qkv), lens, d ** -0.5)
    for more in (4, 8):  # rows of out 8- and 16-byte aligned
        out = torch.full((hq, T + spare, d + more), NAN, dtype=torch.bfloat16, device=DEV)
        lse = torch.full((T + spare, hq + 3), NAN, device=DEV)
        lib.gqa_prompt(q, k, v, i32(cumulative(lens)), d ** -0.5, out[..., :d].transpose(0, 1), lse[:, :hq])
        torch.cuda.synchronize()
        check(out[:, :T, :d].transpose(0, 1), lse[:T, :hq], ref)
        assert out[:, T:].isnan().all() and out[..., d:].isnan().all() and lse[T:].isnan().all() and lse[:, hq:].isnan().all()


@pytest.mark.parametrize("dim,heads", [(64, (64, 64)), (128, (48, 48)), (128, (96, 32))])
def test_many_blocks(dim, heads):
    """More blocks than the chip holds at once: as a prompt, and as chunks whose pages end inside a stage."""
    gen = torch.Generator().manual_seed(dim)
    lens = [1500, 1, 290, 33, 1100]
    q, k, v = randn(gen, sum(lens), heads[0], dim), randn(gen, sum(lens), heads[1], dim), randn(gen, sum(lens), heads[1], dim)
    out, lse = run_prompt(q, k, v, lens, dim ** -0.5)
    check(out, lse, R.prompt(q, k, v, lens, dim ** -0.5))
    c = Paged(lens, [300, 5000, 0, 77, 64], *heads, dim, 16, seed=dim)
    check(*c.run(), c.ref())


@pytest.mark.parametrize("heads,page_size", [((51, 17), 1)])
def test_blocks_of_256_rows(heads, page_size):
    """Long requests that fill the chip with wide blocks; the largest prefix passes the looked-up window of rows."""
    gen = torch.Generator().manual_seed(heads[0])
    lens = [2600]
    q, k, v = randn(gen, sum(lens), heads[0], 128), randn(gen, sum(lens), heads[1], 128), randn(gen, sum(lens), heads[1], 128)
    out, lse = run_prompt(q, k, v, lens, 0.1)
    check(out, lse, R.prompt(q, k, v, lens, 0.1))
    c = Paged([1600, 1000], [3500, 40], *heads, 128, page_size, seed=heads[0])
    check(*c.run(), c.ref())


@pytest.mark.parametrize("page_size", [1, 2, 16, 32, 64, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunk_pages(page_size, dim):
    """Chunks whose pages end inside a tile, at the lengths around tiles and blocks."""
    c = Paged([1, 40, 128, 77], [0, 33, 500, 1030], 8, 2, dim, page_size, seed=page_size + dim)
    check(*c.run(), c.ref())


@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (12, 3), (14, 2), (28, 4), (32, 2), (64, 1)])
@pytest.mark.parametrize("extends", [[1, 1, 1], [3, 1, 2], [9, 4, 16], [70, 1, 33]])
def test_chunk_groups(heads, extends):
    """Every number of rows a request: the stream kernel's 16, 32 and 64, and the blocks of 128."""
    c = Paged(extends, [700, 15, 64], *heads, 128, 16, seed=heads[0] + extends[0])
    check(*c.run(), c.ref())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[1], [2, 31, 32, 33, 127, 128, 129], [5000], [1, 9000, 300], [257] * 70, [300, 1, 512], [700] * 70 + [1024, 3] * 40])
def test_decode_lengths(dim, lens):
    c = Paged([1] * len(lens), [n - 1 for n in lens], 8, 2, dim, 16, seed=len(lens) + lens[0])
    ref = c.ref()
    check(*c.decode(), ref)
    check(*c.run(), ref, "as a chunk")


@pytest.mark.parametrize("extends, prefixes", [
    ([1] * 100, [2999, 4] * 50),  # pieces that fit the CTAs running at once
    ([1] * 301, [1499, 1] * 150 + [8999]),  # many pairs
    ([3, 2, 0] * 30, [2000, 7, 40] * 30),
    ([20, 1] * 40, [1500, 90] * 40),  # blocks
])
def test_split_keys_of_more_requests_than_a_wave_has_lanes(extends, prefixes):
    c = Paged(extends, prefixes, 8, 2, 64, 16, seed=len(extends))
    check(*c.run(), c.ref())


@pytest.mark.parametrize("heads", [(16, 2), (64, 4)])
def test_chunk_long_prefix(heads):
    """Few rows on long prefixes: keys are split and joined, in both kernels, a piece that ends inside a chunk's
    causal end included."""
    c = Paged([3, 1], [6000, 2100], *heads, 128, 64, seed=8)
    check(*c.run(), c.ref(), "streamed")
    c = Paged([150, 1], [5000, 300], *heads, 128, 64, seed=9)
    check(*c.run(), c.ref(), "in blocks")


def test_no_keys_and_no_queries():
    """Requests of no keys (out 0, lse -inf), of no new tokens, and a chunk longer than its keys, whose first queries
    have none."""
    c = Paged([1, 1, 1], [9, 20, 3], 4, 2, 64, 16, seed=4)
    c.lens = [0, 21, 4]
    out, lse = c.run()
    check(out, lse, c.ref())
    assert (out[0] == 0).all() and (lse[0] == -float("inf")).all()
    c = Paged([0, 5, 0, 2, 0], [30, 8, 0, 0, 7], 4, 2, 128, 16, seed=6)
    check(*c.run(), c.ref())
    for rows in (5, 200):
        c = Paged([rows, 3], [40, 3], 4, 1, 64, 16, seed=7)
        c.lens = [rows - 3, 2]
        out, lse = c.run()
        check(out, lse, c.ref())
        assert (out[:3] == 0).all() and (lse[:3] == -float("inf")).all()


def test_rows_behind_the_last_request():
    """A padded batch: rows behind cu_seqlens_q[-1] keep what they hold."""
    for extends in ([1, 2], [150, 30]):
        c = Paged(extends, [100, 40], 8, 2, 128, 16, seed=12, spare_rows=37)
        out, lse = c.run()
        check(out[: c.T], lse[: c.T], c.ref())
        assert out[c.T :].isnan().all() and lse[c.T :].isnan().all()


def test_large_and_far_scores():
    """Scores in the hundreds, whose largest comes last, and a first tile far below: the running maximum moves."""
    for extends, prefixes in (([1, 2], [300, 64]), ([140], [200])):
        c = Paged(extends, prefixes, 8, 2, 128, 16, seed=13, scale=3.0)
        L = c.lens[0]
        rows = c.pt[0].long()[torch.arange(L) // 16] * 16 + torch.arange(L) % 16
        ramp = torch.linspace(0.01, 2.0, L)[:, None, None]
        k = c.k.view(-1, 2, 128)
        k[rows] = (k[rows].float() * ramp).to(torch.bfloat16)
        check(*c.run(), c.ref())


def test_scores_of_minus_infinity():
    """Keys of -inf under positive queries score -inf: they weigh nothing, in a first tile too."""
    for extends in ([1], [140]):
        c = Paged(extends, [200], 4, 2, 64, 16, seed=14)
        c.q = c.q.abs() + 0.1
        rows = c.pt[0].long()[torch.arange(70) // 16] * 16 + torch.arange(70) % 16
        finite = c.k.clone()
        c.k.view(-1, 2, 64)[rows] = -float("inf")
        out, lse = c.run()
        finite.view(-1, 2, 64)[rows] = -1000.0  # scores below exp's range: the same weights
        check(out, lse, R.chunk(c.q, finite, c.v, c.pt, c.extends, c.lens, c.scale)._replace(out_bound=c.ref_bound(finite), lse_bound=torch.tensor(1e-4)))


def _ref_bound(self, k):
    """Bounds that leave out the size of the keys that weigh nothing."""
    k = k.clone()
    k.clamp_(-10, 10)
    return R.chunk(self.q, k, self.v, self.pt, self.extends, self.lens, self.scale).out_bound + 2.0 ** -8 * 4


Paged.ref_bound = _ref_bound


def test_values_that_are_nan_stay_in_their_request():
    """A NaN among a request's keys reaches that request's rows alone."""
    c = Paged([2, 2], [60, 90], 4, 2, 128, 16, seed=15)
    ref = c.ref()
    c.k[int(c.pt[0, 0]), 0] = NAN
    out, lse = c.run()
    assert out[:2].isnan().all() and lse[:2].isnan().all()
    for x, y in zip((out[2:], lse[2:]), (ref.out[2:], ref.lse[2:])):
        assert (x.double().cpu() - y).abs().max() < 0.05


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [NAN, float("inf"), -float("inf")])
def test_later_tokens_that_are_not_finite_reach_no_earlier_row(dim, value):
    """The last tokens' K and V are NaN or infinite: the queries before them are as without them, in one piece and in
    several (a piece that no early query reaches included); those that attend them are not finite."""
    gen = torch.Generator().manual_seed(23)
    lens = [200, 70]
    q, k, v = (randn(gen, sum(lens), h, dim) for h in (6, 2, 2))
    ref = R.prompt(q, k, v, lens, 0.1)
    last = [198, 199, 269]
    keep = [i for i in range(270) if i not in last]
    for t in (k, v):
        t[last] = value
    out, lse = run_prompt(q, k, v, lens, 0.1)
    check(out[keep], lse[keep], R.Attention(*(x[keep] for x in ref)))
    assert not out[last].isfinite().any(-1).all(-1).any()
    for extends, prefixes, heads in (([4, 2], [40, 2000], (6, 2)), ([4, 2], [300, 100], (6, 2)), ([90, 2], [3000, 40], (6, 2)), ([20], [1300], (4, 1)), ([20], [900], (8, 2))):
        c = Paged(extends, prefixes, *heads, dim, 16, seed=24)
        ref = c.ref()
        at = int(c.pt[0, (c.lens[0] - 1) // 16]) * 16 + (c.lens[0] - 1) % 16
        c.v.view(-1, heads[1], dim)[at] = value
        out, lse = c.run()
        keep = [i for i in range(c.T) if i != extends[0] - 1]
        check(out[keep], lse[keep], R.Attention(*(x[keep] for x in ref)), f"{extends} on {prefixes}")
        assert not out[extends[0] - 1].isfinite().any()


@pytest.mark.parametrize("extends,pad", [([1, 1], 0), ([160, 20], 0), ([160, 20], 16384 // 16 + 128)])
def test_pool_past_32_bits(extends, pad):
    """K and V rows past 2^31 bytes and 2^31 elements from the pool's start; with rows behind the requests, in blocks."""
    pages, ps, hk, d = 17000, 64, 8, 128  # 1.1 G elements a pool, 2.2 GB
    gen = torch.Generator(device=DEV).manual_seed(0)
    k = torch.empty((2 * pages, ps, hk, d), dtype=torch.bfloat16, device=DEV)
    v = torch.empty_like(k)
    used = [2 * pages - 1, 0, pages, pages - 1, 2 * pages - 2, 3, 2 * pages - 5, 7]
    for p in used:
        k[p] = torch.randn(k[p].shape, generator=gen, device=DEV).to(torch.bfloat16)
        v[p] = torch.randn(k[p].shape, generator=gen, device=DEV).to(torch.bfloat16)
    pt = torch.tensor([used[:4], used[4:]], dtype=torch.int32)
    lens, T = [250, 256], sum(extends)
    q = torch.randn((T + pad, 16, d), generator=gen, device=DEV).to(torch.bfloat16)
    out, lse = torch.empty_like(q), torch.empty((T + pad, 16), device=DEV)
    lib.gqa_chunk(q, k, v, pt.to(DEV), i32(cumulative(extends)), i32(lens), max(extends) + pad, d ** -0.5, out, lse)
    torch.cuda.synchronize()
    index = torch.tensor(used, device=DEV)
    small = torch.tensor([[0, 1, 2, 3], [4, 5, 6, 7]], dtype=torch.int32)
    check(out[:T], lse[:T], R.chunk(q[:T].cpu(), k[index].cpu(), v[index].cpu(), small, extends, lens, d ** -0.5))


def test_device_lengths_and_page_ids_out_of_range_are_cut():
    """Lengths past the page table and page ids outside the pool are cut and clamped: the call reads its tensors alone."""
    c = Paged([1, 130], [40, 100], 4, 2, 64, 16, seed=16)
    c.k.nan_to_num_(0.5), c.v.nan_to_num_(0.5)
    c.pt[0, 0], c.pt[1, 1] = 10 ** 6, -5
    lens, pages = list(c.lens), c.k.shape[0]
    c.lens = [40 + 1, 10 ** 9]
    out, lse = c.run()
    c.pt.clamp_(0, pages - 1)
    c.lens = [lens[0], c.pt.shape[1] * 16]
    check(out, lse, c.ref())


@pytest.mark.parametrize("extends,prefixes", [([1] * 5, [3000, 10, 700, 1, 90]), ([200, 3], [3000, 10])])
def test_capture_and_replay_with_other_lengths(extends, prefixes):
    """A captured call follows the lengths and tables of each replay, next to eager calls of its own."""
    a = Paged(extends, prefixes, 8, 2, 128, 16, seed=17)
    cu = i32(cumulative(extends))
    q, k, v, pt, lens = a.q.to(DEV), a.k.to(DEV), a.v.to(DEV), a.pt.to(DEV), i32(a.lens)
    ws = lib.gqa_workspace(max(extends), 8, 2, 128, DEV)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device=DEV)
    call = lambda: lib.gqa_chunk(q, k, v, pt, cu, lens, max(extends), a.scale, out, lse, ws)  # noqa: E731
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for cut in (0, 5, 2, 0):
        new = [max(n - cut * 37, e) for n, e in zip(a.lens, extends)]
        lens.copy_(i32(new))
        out.fill_(NAN), lse.fill_(NAN)
        graph.replay()
        got = out.clone(), lse.clone()
        other = Paged([1, 7], [50, 60], 8, 2, 128, 16, seed=18)
        check(*other.run(), other.ref(), "eager, between replays")
        ref = R.chunk(a.q, a.k, a.v, a.pt, extends, new, a.scale)
        check(*got, ref, f"replay with lengths {new}")
        out.fill_(NAN), lse.fill_(NAN)
        call()
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], lse), "replay and eager call differ"


@pytest.mark.parametrize("extends", [[1, 1], [5, 8], [16, 3], [300, 1]])
def test_one_workspace_for_steps_of_all_sizes(extends):
    c = Paged(extends, [4000, 2500], 8, 1, 128, 16, seed=sum(extends))
    out, lse = c.run(workspace=lib.gqa_workspace(300, 8, 1, 128, DEV))
    check(out, lse, c.ref())


def test_captured_calls_without_a_workspace():
    """Two graphs whose split keys use memory of their own pools, replayed in turn with eager calls and allocations between."""
    made = []
    for seed, extends, prefixes in ((31, [1, 1, 1], [3000, 40, 5000]), (32, [200, 3], [4000, 10])):
        c = Paged(extends, prefixes, 8, 2, 128, 16, seed=seed)
        cu, lens = i32(cumulative(extends)), i32(c.lens)
        dev = [x.to(DEV) for x in (c.q, c.k, c.v, c.pt)]
        out, lse = torch.empty_like(dev[0]), torch.empty(c.q.shape[:2], device=DEV)
        call = lambda dev=dev, cu=cu, lens=lens, n=max(extends), s=c.scale, out=out, lse=lse: lib.gqa_chunk(*dev, cu, lens, n, s, out, lse)  # noqa: E731
        call()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call()
        made.append((graph, out, lse, c.ref(), call))  # which holds the inputs
    for _ in range(3):
        for graph, out, lse, ref, _ in made:
            out.fill_(NAN), lse.fill_(NAN)
            graph.replay()
            junk = torch.full((1 << 25,), NAN, device=DEV)
            other = Paged([1, 7], [3000, 60], 8, 2, 128, 16, seed=33)
            check(*other.run(), other.ref(), "eager, between replays")
            check(out, lse, ref)
            del junk


def padding(q_heads):
    """Rows behind the last request that make a batch one of more 16-row CTAs than run at once: its kernel is the blocks'."""
    return 16384 // q_heads + 128


class InBlocks(Paged):
    """A small batch that takes the kernel of the large ones."""

    def __init__(self, extends, prefixes, q_heads, *args, **kw):
        super().__init__(extends, prefixes, q_heads, *args, spare_rows=padding(q_heads), **kw)

    def run(self, workspace=None):
        out, lse = super().run(self.q.shape[0], workspace)
        assert out[self.T :].isnan().all() and lse[self.T :].isnan().all()
        return out[: self.T], lse[: self.T]


def prompt_in_blocks(q, k, v, lens, scale):
    T, pad = q.shape[0], padding(q.shape[1])
    out, lse = run_prompt(*(torch.cat((x, torch.full((pad, *x.shape[1:]), NAN, dtype=x.dtype))) for x in (q, k, v)), lens, scale)
    assert out[T:].isnan().all() and lse[T:].isnan().all()
    return out[:T], lse[:T]


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("heads", [(1, 1), (8, 1), (4, 4), (6, 2), (14, 2), (20, 4), (48, 3)])
def test_prompt_heads_in_blocks(dim, heads):
    gen = torch.Generator().manual_seed(heads[0] * dim)
    lens = [33, 1, 0, 129, 64]
    q, k, v = randn(gen, sum(lens), heads[0], dim), randn(gen, sum(lens), heads[1], dim), randn(gen, sum(lens), heads[1], dim)
    check(*prompt_in_blocks(q, k, v, lens, dim ** -0.5), R.prompt(q, k, v, lens, dim ** -0.5))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[1], [31, 32, 33], [127, 128, 129], [255, 257], [1500, 3, 700], [2, 17, 1, 0, 40] * 30])
def test_prompt_lengths_in_blocks(dim, lens):
    gen = torch.Generator().manual_seed(sum(lens))
    q, k, v = randn(gen, sum(lens), 4, dim), randn(gen, sum(lens), 2, dim), randn(gen, sum(lens), 2, dim)
    check(*prompt_in_blocks(q, k, v, lens, dim ** -0.5), R.prompt(q, k, v, lens, dim ** -0.5))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens,heads", [([150, 30, 300, 1, 200, 90, 20, 0, 250, 50], (8, 2)), ([60] * 9, (16, 4)), ([550], (17, 17)), ([1] * 40, (30, 15))])
def test_prompts_between_few_ctas_and_blocks(dim, lens, heads):
    """16-row CTAs that run at once, four waves each."""
    gen = torch.Generator().manual_seed(len(lens))
    q, k, v = randn(gen, sum(lens), heads[0], dim), randn(gen, sum(lens), heads[1], dim), randn(gen, sum(lens), heads[1], dim)
    out, lse = run_prompt(q, k, v, lens, dim ** -0.5)
    check(out, lse, R.prompt(q, k, v, lens, dim ** -0.5))
    c = Paged([n % 61 for n in lens], [n // 2 for n in lens], *heads, dim, 16, seed=len(lens))
    check(*c.run(), c.ref())


@pytest.mark.parametrize("dim,lens,heads", [(64, [2100], (6, 2)), (64, [1300], (12, 2)), (64, [3001, 70], (4, 4)), (128, [2049], (10, 5)), (128, [4100], (4, 1))])
@pytest.mark.parametrize("value", [None, NAN, float("inf")])
def test_long_prompts_on_few_heads(dim, lens, heads, value):
    """Blocks alone on their compute units, the first of them without keys in the second half; later tokens that are not
    finite."""
    gen = torch.Generator().manual_seed(lens[0])
    q, k, v = randn(gen, sum(lens), heads[0], dim), randn(gen, sum(lens), heads[1], dim), randn(gen, sum(lens), heads[1], dim)
    ref = R.prompt(q, k, v, lens, 0.1)
    keep = list(range(sum(lens)))
    if value is not None:
        last = [lens[0] - 1, lens[0] - 40]
        v[last] = value
        keep = [i for i in keep if not lens[0] - 40 <= i < lens[0]]
    out, lse = run_prompt(q, k, v, lens, 0.1)
    check(out[keep], lse[keep], R.Attention(*(x[keep] for x in ref)))
    if value is not None:
        assert not out[lens[0] - 40 : lens[0]].isfinite().any()


@pytest.mark.parametrize("page_size", [1, 2, 16, 32, 256])
@pytest.mark.parametrize("dim", [64, 128])
def test_chunk_pages_in_blocks(page_size, dim):
    for prefixes in ([0, 33, 500, 1030], [0, 33, 500, 30]):  # keys split, and in one piece
        c = InBlocks([1, 40, 128, 77], prefixes, 8, 2, dim, page_size, seed=page_size + dim)
        check(*c.run(), c.ref())


@pytest.mark.parametrize("heads", [(1, 1), (8, 8), (12, 3), (14, 2), (28, 4), (64, 1)])
@pytest.mark.parametrize("extends", [[1, 1, 1], [9, 4, 16], [70, 1, 33]])
def test_chunk_groups_in_blocks(heads, extends):
    c = InBlocks(extends, [700, 15, 64], *heads, 128, 16, seed=heads[0] + extends[0])
    check(*c.run(), c.ref())


def test_no_keys_and_far_scores_in_blocks():
    c = InBlocks([0, 5, 0, 2, 0], [30, 8, 0, 0, 7], 4, 2, 128, 16, seed=6)
    check(*c.run(), c.ref())
    c = InBlocks([200, 3], [40, 3], 4, 1, 64, 16, seed=7)
    c.lens = [197, 2]
    out, lse = c.run()
    check(out, lse, c.ref())
    assert (out[:3] == 0).all() and (lse[:3] == -float("inf")).all()
    c = InBlocks([140], [200], 8, 2, 128, 16, seed=13, scale=3.0)
    rows = c.pt[0].long()[torch.arange(340) // 16] * 16 + torch.arange(340) % 16
    k = c.k.view(-1, 2, 128)
    k[rows] = (k[rows].float() * torch.linspace(0.01, 2.0, 340)[:, None, None]).to(torch.bfloat16)
    check(*c.run(), c.ref())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("value", [NAN, float("inf"), -float("inf")])
def test_later_tokens_that_are_not_finite_in_blocks(dim, value):
    gen = torch.Generator().manual_seed(23)
    lens, last = [200, 70], [198, 199, 269]
    q, k, v = (randn(gen, sum(lens), h, dim) for h in (6, 2, 2))
    ref = R.prompt(q, k, v, lens, 0.1)
    keep = [i for i in range(270) if i not in last]
    for t in (k, v):
        t[last] = value
    out, lse = prompt_in_blocks(q, k, v, lens, 0.1)
    check(out[keep], lse[keep], R.Attention(*(x[keep] for x in ref)))
    assert not out[last].isfinite().any(-1).all(-1).any()
    for extends, prefixes in (([90, 2], [3000, 40]), ([20, 40], [300, 2])):
        c = InBlocks(extends, prefixes, 6, 2, dim, 16, seed=24)
        ref = c.ref()
        at = int(c.pt[0, (c.lens[0] - 1) // 16]) * 16 + (c.lens[0] - 1) % 16
        c.v.view(-1, 2, dim)[at] = value
        out, lse = c.run()
        keep = [i for i in range(c.T) if i != extends[0] - 1]
        check(out[keep], lse[keep], R.Attention(*(x[keep] for x in ref)))


def test_device_lengths_and_page_ids_out_of_range_are_cut_in_blocks():
    c = InBlocks([1, 130], [40, 100], 4, 2, 64, 16, seed=16)
    c.k.nan_to_num_(0.5), c.v.nan_to_num_(0.5)
    c.pt[0, 0], c.pt[1, 1] = 10 ** 6, -5
    c.lens = [41, 10 ** 9]
    out, lse = c.run()
    c.pt.clamp_(0, c.k.shape[0] - 1)
    c.lens = [41, c.pt.shape[1] * 16]
    check(out, lse, c.ref())


def test_two_streams_with_workspaces_of_their_own():
    a, b = (Paged([2, 1], [4000, 900], 8, 2, 128, 16, seed=s) for s in (19, 20))
    streams = [torch.cuda.Stream() for _ in range(2)]
    made = []
    for c, s in zip((a, b), streams):
        dev = [t.to(DEV) for t in (c.q, c.k, c.v, c.pt)] + [i32(cumulative(c.extends)), i32(c.lens)]
        made.append((dev, torch.full_like(dev[0], NAN), torch.full(c.q.shape[:2], NAN, device=DEV), lib.gqa_workspace(2, 8, 2, 128, DEV)))
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s, ((q, k, v, pt, cu, lens), out, lse, ws) in zip((a, b), streams, made):
            lib.gqa_chunk(q, k, v, pt, cu, lens, 2, c.scale, out, lse, ws, stream=s)
    torch.cuda.synchronize()
    for c, (_, out, lse, _) in zip((a, b), made):
        check(out, lse, c.ref())


def test_repeated_calls_are_bit_equal():
    """No order of arrival enters a result."""
    for extends, prefixes in (([1, 1, 1], [5000, 40, 700]), ([150, 2], [3000, 9])):
        c = Paged(extends, prefixes, 16, 2, 128, 16, seed=21)
        first = c.run()
        for _ in range(4):
            again = c.run()
            assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_decode_without_lse():
    c = Paged([1, 1], [600, 20], 8, 2, 128, 16, seed=22)
    q = c.q.to(DEV)
    out = torch.empty_like(q)
    lib.gqa_decode(q, c.k.to(DEV), c.v.to(DEV), c.pt.to(DEV), i32(c.lens), c.scale, out)
    assert torch.equal(out, c.decode()[0])
