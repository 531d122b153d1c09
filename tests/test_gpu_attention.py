"""Attention of one new token a sequence over a paged cache on the GPU against its
definition in float64 (tests/layer_ref.py, where the tolerances are derived).

Unless a test says otherwise, everything that a call must not look at is NaN: the
places behind each sequence's length, the pages of no sequence, what lies before a
window; page numbers behind a sequence are out of range."""
import numpy as np
import pytest
import torch

from gollek_amd import _native
from gollek_amd import tensor_ops as ops
from tests import layer_ref as ref
from tests.layer_ref import BF16, DTYPE, F16, F32
from tests.test_gpu_layer_ops import close, normal, ptr, rng, stream

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def _init():
    ops.init(0)


class Batch:
    """A cache of sequences of the given lengths, and one query row for each."""

    def __init__(self, lengths, q_heads, kv_heads, dim, cache_type=BF16, *, page=16, window=0, max_pages=None, seed=0,
                 q_sigma=2.0, k_sigma=1.0):
        g = self.g = rng(seed)
        self.lengths, self.q_heads, self.kv_heads, self.dim, self.page = list(lengths), q_heads, kv_heads, dim, page
        self.type, self.window = cache_type, window
        n = len(lengths)
        need = [-(-max(x, 0) // page) for x in lengths]
        self.max_pages = max(need + [1]) if max_pages is None else max_pages
        pool = sum(need) + 2
        order = torch.randperm(pool, generator=g).to(torch.int32)
        table = torch.full((n, self.max_pages), -1, dtype=torch.int32)
        table[1::2] = 2**31 - 1
        k = torch.full((pool, kv_heads, page, dim), float("nan"))
        v = torch.full((pool, kv_heads, page, dim), float("nan"))
        at = 0
        for s, length in enumerate(lengths):
            begin = max(0, length - window) if window else 0
            for c in range(need[s]):
                number = int(order[at])
                at += 1
                if (c + 1) * page <= begin:
                    continue  # before the window: no page at all
                table[s, c] = number
                first, last = max(begin - c * page, 0), min(page, length - c * page)
                k[number, :, first:last] = normal(g, kv_heads, last - first, dim, sigma=k_sigma)
                v[number, :, first:last] = normal(g, kv_heads, last - first, dim)
        self.table, self.k, self.v = table, k.to(DTYPE[cache_type]), v.to(DTYPE[cache_type])
        self.q = normal(g, n, q_heads, dim, sigma=q_sigma).to(DTYPE[cache_type])
        self.device()

    def device(self):
        self.dk, self.dv, self.dq, self.dt = self.k.cuda(), self.v.cuda(), self.q.cuda(), self.table.cuda()
        self.dl = torch.tensor(self.lengths, dtype=torch.int32).cuda()
        self.cache = ops.KvCache(self.type, ptr(self.dk), ptr(self.dv), self.dk.shape[0], self.page, self.kv_heads, self.dim)
        self.need = self.cache.attend_workspace_bytes(len(self.lengths), self.q_heads, self.max_pages)
        self.ws = torch.full((self.need + 256,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN
        return self

    def attend(self, out_type=F32, *, scale=None, softcap=0.0, sinks=None, q=None, q_stride=0, out=None, out_stride=0, on=None):
        n = len(self.lengths)
        scale = ref.softmax_scale(self.dim) if scale is None else scale
        if out is None:
            out = torch.full((n, self.q_heads, self.dim), float("nan"), dtype=DTYPE[out_type], device="cuda")
        print(f"[gpu] attend lengths={self.lengths[:8]} of {n} heads={self.q_heads}/{self.kv_heads}x{self.dim} "
              f"type={self.type}->{out_type} page={self.page} window={self.window}", flush=True)
        self.cache.attend(ptr(self.dq if q is None else q), n, self.q_heads, ptr(self.dl), ptr(self.dt), self.max_pages, ptr(out),
                          out_type, scale=scale, softcap=softcap, window=self.window, sinks_ptr=ptr(sinks), q_stride=q_stride,
                          out_stride=out_stride, ws_ptr=ptr(self.ws), ws_bytes=self.need, stream=stream() if on is None else on)
        return out

    def check(self, out_type=F32, rows=None, **kw):
        out = self.attend(out_type, **kw)
        torch.cuda.synchronize()
        assert torch.all(self.ws[self.need:] == 0xFF)
        self.compare(out, out_type, rows, **kw)
        return out

    def compare(self, out, out_type, rows=None, *, scale=None, softcap=0.0, sinks=None, **_):
        scale = ref.softmax_scale(self.dim) if scale is None else scale
        for s in range(len(self.lengths)) if rows is None else rows:
            length = min(max(self.lengths[s], 0), self.max_pages * self.page)
            begin = max(0, length - self.window) if self.window else 0
            at = np.arange(begin, length)
            numbers = self.table[s].numpy()[at // self.page]
            good = (numbers >= 0) & (numbers < self.k.shape[0])
            where = (torch.from_numpy(numbers[good].astype(np.int64)), slice(None), torch.from_numpy(at[good] % self.page))
            want, off = ref.attention(self.q[s], self.k[where], self.v[where], scale=scale, softcap=softcap, sinks=sinks)
            close(out[s], want, off, out_type, f"sequence {s} of length {length}")


EDGES = [0, 1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 255, 257, 500]


@pytest.mark.parametrize("cache_type", [F16, BF16])
@pytest.mark.parametrize("out_type", [F32, F16, BF16])
def test_lengths_and_types(cache_type, out_type):
    Batch(EDGES, 8, 2, 128, cache_type, seed=1).check(out_type)


@pytest.mark.parametrize("dim", [8, 16, 24, 32, 40, 64, 72, 80, 96, 104, 112, 128, 136, 160, 192, 200, 224, 256])
def test_head_dims(dim):
    Batch([0, 1, 17, 50, 130], 4, 2, dim, BF16, seed=dim).check(F32)
    Batch([33, 7], 2, 2, dim, F16, seed=dim).check(F16)


@pytest.mark.parametrize("q_heads,kv_heads", [(1, 1), (2, 1), (3, 1), (7, 1), (8, 8), (10, 2), (16, 1), (17, 1), (32, 2), (40, 1),
                                              (64, 8), (71, 1), (128, 1)])
def test_head_groups(q_heads, kv_heads):
    Batch([0, 5, 90, 200], q_heads, kv_heads, 64, BF16, seed=q_heads).check(F32)


@pytest.mark.parametrize("page", [16, 32, 64, 256, 4096])
def test_page_sizes(page):
    Batch([1, 16, 40, 300, 1000], 8, 2, 64, F16, page=page, seed=page).check(F32)
    Batch([1, 40, 300], 8, 2, 64, F16, page=page, window=37, seed=page).check(F32)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 128, 4096])
@pytest.mark.parametrize("page", [16, 64])
def test_windows(window, page):
    Batch([0, 1, 16, 17, 100, 128, 129, 145, 600], 8, 2, 64, BF16, page=page, window=window, seed=window).check(F32)


@pytest.mark.parametrize("softcap", [0.5, 30.0, 50.0])
def test_softcap(softcap):
    Batch([0, 1, 77, 400], 4, 1, 64, BF16, seed=6).check(F32, softcap=softcap)


def test_sinks():
    b = Batch([0, 1, 77, 400], 16, 2, 64, F16, seed=7)
    for values in (normal(rng(8), 16, sigma=3.0), torch.full((16,), -float("inf")), torch.full((16,), 60.0)):
        b.check(F32, sinks=values.cuda())
    b = Batch([0, 1, 77, 400], 16, 2, 64, F16, window=20, seed=7)
    b.check(BF16, sinks=normal(rng(8), 16, sigma=3.0).cuda(), softcap=20.0)


@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0])
def test_scales(scale):
    Batch([1, 50, 300], 4, 2, 64, BF16, q_sigma=1.0, seed=9).check(F32, scale=scale)


def test_sharp_and_flat_rows():
    # scores of hundreds: a row is one token; scores of nothing: a mean over all
    Batch([3, 700, 2100], 8, 1, 128, F16, q_sigma=30.0, seed=10).check(F32, scale=0.5)
    Batch([3, 700, 2100], 8, 1, 128, F16, q_sigma=0.01, seed=11).check(F32)
    Batch([3, 700, 2100], 8, 1, 128, BF16, q_sigma=0.01, seed=12).check(F32)


def test_weights_far_below_the_largest_add_up():
    # one token of score 0, 4000 of -12 to -10: together 4 % of the sum, each below fp16's normal numbers
    b = Batch([4001], 4, 1, 64, F16, seed=13)
    b.q.fill_(1.0)
    rows = (b.table[0].numpy()[np.arange(4001) // 16], np.arange(4001) % 16)
    b.k[torch.from_numpy(rows[0].astype(np.int64)), 0, torch.from_numpy(rows[1])] = (-torch.linspace(10, 12, 4001)[:, None] / 64).expand(4001, 64).half()
    b.k[int(rows[0][0]), 0, 0] = 0.0
    b.v.abs_()
    b.device().check(F32, scale=1.0)
    b.check(F16, scale=1.0)


@pytest.mark.parametrize("lengths,q_heads,kv_heads,dim", [([40000], 8, 1, 128), ([20011], 32, 8, 64), ([9000, 3], 4, 4, 128),
                                                          ([16384, 1, 700, 0, 5000], 16, 2, 128)])
def test_long_sequences(lengths, q_heads, kv_heads, dim):
    Batch(lengths, q_heads, kv_heads, dim, BF16, seed=14).check(F32)
    Batch(lengths, q_heads, kv_heads, dim, F16, window=3000, seed=15).check(BF16)


def test_many_sequences():
    lengths = [(37 * i) % 211 for i in range(300)]
    Batch(lengths, 8, 2, 64, BF16, seed=16).check(F32)
    Batch([(5 * i) % 9 for i in range(3000)], 2, 1, 32, BF16, seed=17).check(F32)


@pytest.mark.parametrize("sequences,kv_heads,dim", [(50, 8, 128), (50, 8, 256), (50, 8, 40), (20, 8, 128), (3, 1, 256), (2, 1, 8),
                                                    (97, 16, 64), (300, 2, 192), (1024, 1, 64), (1025, 1, 64)])
def test_few_long_among_many(sequences, kv_heads, dim):
    # every way to join chunks: many a sequence, a few, at most one on the average
    lengths = [(11 * i) % 67 for i in range(sequences)]
    lengths[0], lengths[sequences // 2], lengths[-1] = 3000, 1111, 5000
    rows = sorted({0, 1, sequences // 3, sequences // 2, sequences - 2, sequences - 1})
    Batch(lengths, 2 * kv_heads, kv_heads, dim, BF16, page=64, seed=sequences).check(F32, rows)


@pytest.mark.parametrize("q_heads,kv_heads,dim", [(16, 8, 64), (8, 8, 128), (24, 8, 80), (8, 8, 256), (16, 8, 192), (136, 8, 40),
                                                  (32, 8, 24), (8, 8, 8)])
@pytest.mark.parametrize("cache_type,out_type", [(BF16, F32), (F16, BF16), (BF16, F16)])
def test_many_short_sequences(q_heads, kv_heads, dim, cache_type, out_type):
    # enough heads of so few tokens that each is a wave's
    sequences = 260
    lengths = [(13 * i) % 150 for i in range(sequences)]
    rows = [0, 1, 2, 5, 11, 12, 23, 100, 101, 258, 259]
    b = Batch(lengths, q_heads, kv_heads, dim, cache_type, page=32, seed=dim)
    b.check(out_type, rows)
    b.check(out_type, rows, sinks=normal(rng(dim), q_heads, sigma=2.0).cuda(), softcap=10.0)
    b = Batch([7 * x for x in lengths], q_heads, kv_heads, dim, cache_type, page=16, window=100, seed=dim)
    b.table[11, 2 * 11] = -1
    b.device().check(out_type, rows)


@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("most", [9, 60, 180, 300, 340])
def test_short_sequences_around_the_rules(dim, most):
    # units on both sides of the border between a workgroup and a wave each
    for sequences in (63, 64, 95, 96, 127, 128, 160, 192):
        lengths = [(29 * i) % (most + 1) for i in range(sequences)]
        lengths[-1] = most
        Batch(lengths, 8, 8, dim, BF16, page=64, seed=dim + sequences).check(BF16, [0, 1, sequences // 2, sequences - 1])


def test_many_short_sequences_in_strided_rows():
    lengths = [(13 * i) % 90 for i in range(1030)]
    b = Batch(lengths, 4, 2, 64, BF16, seed=33)
    for out_type, shift in ((F32, 1), (BF16, 3), (F16, 8)):
        out = torch.full((1030 * 301 + 8,), float("nan"), dtype=DTYPE[out_type], device="cuda")
        b.attend(out_type, out=out[shift:], out_stride=301)
        torch.cuda.synchronize()
        rows = out[shift:shift + 1030 * 301].view(1030, 301)
        b.compare(rows[:, :256].reshape(1030, 4, 64), out_type, range(0, 1030, 41))
        assert torch.isnan(rows[:, 256:]).all() and torch.isnan(out[:shift]).all() and not torch.isnan(rows[:, :256]).any()


def test_tables_much_wider_than_the_lengths():
    # cut by the lengths, not by the table
    for lengths in ([5, 700, 0], [3000], [0, 0, 0, 0], [0], [1, 2, 3]):
        b = Batch(lengths, 8, 2, 128, BF16, max_pages=5000, seed=34)
        b.check(F32)
        b.check(BF16, sinks=normal(rng(35), 8).cuda())


def test_one_large_page_a_sequence():
    b = Batch([65536, 1, 40001], 4, 1, 64, F16, page=65536, seed=36)
    b.check(F32)
    Batch([65536, 70, 40001], 4, 1, 64, F16, page=65536, window=50, seed=36).check(F32)


@pytest.mark.parametrize("scale,softcap", [(1e15, 1e-15), (1e-15, 1e15), (0.125, 1e15), (0.125, 1e-15)])
def test_extreme_scales(scale, softcap):
    # weights alike, or the largest score's alone: nothing overflows on the way
    b = Batch([40, 300], 4, 2, 64, BF16, seed=37)
    out = b.attend(F32, scale=scale, softcap=softcap)
    torch.cuda.synchronize()
    assert torch.isfinite(out).all()


def test_lengths_past_the_table_and_below_zero():
    b = Batch([64, 64, 64, 64], 4, 2, 64, BF16, seed=18)
    b.lengths = [65, 2**31 - 1, -5, -(2**31)]
    b.device().check(F32)


def test_pages_that_are_none():
    # in the middle, at the start, at the end, all of them
    b = Batch([200, 200, 200, 200, 200], 8, 2, 64, BF16, seed=19)
    b.table[0, 3] = -1
    b.table[1, 0], b.table[1, 1] = 2**31 - 1, -(2**31)
    b.table[2, 12] = b.k.shape[0]
    b.table[3] = -7
    out = b.device().check(F32)
    assert not out[3].any()
    b.check(F32, sinks=normal(rng(20), 8).cuda())


def test_strides_and_what_lies_between():
    b = Batch([30, 0, 77], 4, 2, 64, BF16, seed=21)
    q = torch.full((3, 700), float("nan"), dtype=torch.bfloat16, device="cuda")
    q[:, 3:3 + 256] = b.dq.view(3, 256)  # off every 16-byte border
    for out_type, shift in ((F32, 1), (BF16, 3), (F16, 8)):
        out = torch.full((3 * 301 + 8,), float("nan"), dtype=DTYPE[out_type], device="cuda")
        b.attend(out_type, q=q[:, 3:], q_stride=700, out=out[shift:], out_stride=301)
        torch.cuda.synchronize()
        rows = out[shift:shift + 903].view(3, 301)
        b.compare(rows[:, :256].reshape(3, 4, 64), out_type)
        assert torch.isnan(rows[:, 256:]).all() and torch.isnan(out[:shift]).all() and torch.isnan(out[shift + 903:]).all()


def test_infinities_of_a_key():
    # a key of -inf where the query is positive has no weight; a row of nothing else is NaN or 0, never a wrong number
    b = Batch([40], 2, 1, 64, BF16, seed=22)
    b.q.abs_()
    number, slot = int(b.table[0, 1]), 3
    b.k[number, 0, slot, 5] = -float("inf")
    out = b.device().attend(F32)
    torch.cuda.synchronize()
    without = [j for j in range(40) if j != 19]
    k, v = ref.gather(b.k, b.table[0], 40)[without], ref.gather(b.v, b.table[0], 40)[without]
    want, off = ref.attention(b.q[0], k, v, scale=ref.softmax_scale(64))
    close(out[0], want, off, F32)


def test_nan_of_a_key_stays_in_its_head():
    b = Batch([40, 50], 4, 2, 64, BF16, seed=23)
    b.k[int(b.table[0, 0]), 1, 2, 9] = float("nan")
    out = b.device().attend(F32)
    torch.cuda.synchronize()
    assert torch.isnan(out[0, 2:]).all()
    assert not torch.isnan(out[0, :2]).any() and not torch.isnan(out[1]).any()


def test_same_page_in_two_sequences_and_several_tokens_of_one():
    # a shared prefix, and four new tokens of one sequence as rows of growing lengths
    b = Batch([100, 100, 100, 100], 8, 2, 64, BF16, seed=24)
    b.table[1:] = b.table[0]
    b.lengths = [97, 98, 99, 100]
    b.device().check(F32)


def test_repeats_give_the_same_bits():
    b = Batch([9000, 40, 2500], 16, 2, 128, BF16, seed=25)
    first = b.attend(F32)
    for _ in range(5):
        assert torch.equal(b.attend(F32), first)


def test_two_streams_at_once():
    a, b = Batch([7000, 300], 8, 2, 128, BF16, seed=26), Batch([5000, 10, 900], 8, 1, 64, F16, seed=27)
    want = a.attend(F32).clone(), b.attend(F32).clone()
    torch.cuda.synchronize()
    one, two = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(8):
        outs.append((a.attend(F32, on=one.cuda_stream), b.attend(F32, on=two.cuda_stream)))
    torch.cuda.synchronize()
    for x, y in outs:
        assert torch.equal(x, want[0]) and torch.equal(y, want[1])


def test_captured_and_replayed_with_growing_lengths():
    b = Batch([6000, 90, 1], 8, 2, 64, BF16, seed=28)
    full = list(b.lengths)
    out = torch.empty(3, 8, 64, device="cuda")
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        b.attend(F32, out=out, on=side.cuda_stream)
    for lengths in ([1, 1, 0], [17, 90, 1], [5999, 0, 1], full, [3000, 45, 1], full):
        b.lengths = lengths
        b.dl.copy_(torch.tensor(lengths, dtype=torch.int32))
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        b.compare(replayed, F32)
        assert torch.equal(b.attend(F32), replayed)


def test_graphs_that_share_a_workspace():
    a, b = Batch([4000, 70], 8, 2, 64, BF16, seed=29), Batch([50, 3000, 800], 8, 1, 128, BF16, seed=30)
    if a.need < b.need:
        a.ws = b.ws
    else:
        b.ws = a.ws
    outs = torch.empty(2, 8, 64, device="cuda"), torch.empty(3, 8, 128, device="cuda")
    graphs = []
    side = torch.cuda.Stream()
    for x, out in zip((a, b), outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            x.attend(F32, out=out, on=side.cuda_stream)
        graphs.append(g)
    for _ in range(3):
        for i in (0, 1, 1, 0):
            outs[i].fill_(float("nan"))
            graphs[i].replay()
            (a, b)[i].compare(outs[i], F32)


def test_a_small_call_needs_no_more_than_its_own_workspace():
    b = Batch([40], 4, 2, 64, BF16, seed=31)
    if b.need:
        with pytest.raises(ops.IllegalArgumentError):
            b.cache.attend(ptr(b.dq), 1, 4, ptr(b.dl), ptr(b.dt), b.max_pages, ptr(torch.empty(1, 4, 64, device="cuda")), F32,
                           scale=1.0, ws_ptr=ptr(b.ws), ws_bytes=b.need - 1, stream=stream())
    b.check(F32)
