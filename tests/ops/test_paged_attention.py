"""GPU parity of the paged-cache ops against the 64-bit oracle; values are held to its error bound
plus half a step of their type."""

import math

import pytest
import torch

from oracle import serving_attention as ref
from oracle.recurrent import assert_within
from tileops import _native as nat
from tileops.ops.attention import PagedAttentionDecodeOp, PagedKVAppendOp, rotary_frequencies

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
HALF = [torch.float16, torch.bfloat16]


def _flag(clear=1):
    return nat.lib().tileops_device_error_flag(nat.stream_handle(torch.device("cuda", 0)), clear)


@pytest.fixture(autouse=True)
def no_flag():
    _flag()
    yield
    assert _flag() == 0


def _cache(pages, P, Hkv, D, dtype, layout="token", fill=None):
    shape = (pages, P, Hkv, D) if layout == "token" else (pages, Hkv, P, D)
    c = torch.randn(shape, device="cuda").to(dtype) if fill is None else torch.full(
        shape, fill, device="cuda", dtype=dtype)
    return c if layout == "token" else c.transpose(1, 2)


def _table(lens, P, extra=0, spare=3):
    """Pages of every sequence in a mixed order, -1 behind its end, and how many pages there are."""
    need = [max(0, -(-n // P)) for n in lens]
    width = max([1, *need]) + extra
    order = torch.randperm(sum(need) + spare).tolist()
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for c in range(n):
            table[b, c] = order.pop()
    return table.cuda(), sum(need) + spare


def _lens(lens):
    return torch.tensor(lens, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------ attention
def _whole(*shape, dtype):
    """Whole numbers from -2 to 2: products and sums of them are exact."""
    return torch.randint(-2, 3, shape, device="cuda").to(dtype)


def _attend(lens, H, Hkv, D, P, dtype, layout="token", window=None, scale=None, exact=True, extra=0):
    """Behind each sequence's end (and before its window) the cache holds NaN; the first and last
    tokens that count hold large values, so that one too few shows in o."""
    table, pages = _table(lens, P, extra)
    kc, vc = _cache(pages, P, Hkv, D, dtype, layout, fill=math.nan), _cache(
        pages, P, Hkv, D, dtype, layout, fill=math.nan)
    for b, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        at = torch.arange(first, max(n, 0), device="cuda")
        where = (table[b].long()[at // P], at % P)
        kc[where] = _whole(len(at), Hkv, D, dtype=dtype) if exact else torch.randn(
            len(at), Hkv, D, device="cuda").to(dtype)
        v = torch.randn(len(at), Hkv, D, device="cuda")
        if n > 0:
            v[0] += 50
            v[-1] -= 70
        vc[where] = v.to(dtype)
    q = _whole(len(lens), H, D, dtype=dtype) if exact else (
        2 * torch.randn(len(lens), H, D, device="cuda")).to(dtype)
    scale = 0.25 / D**0.5 if scale is None and exact else scale
    op = PagedAttentionDecodeOp(H, Hkv, D, P, scale, window, dtype)
    lens = _lens(lens)
    o, lse = op(q, kc, vc, table, lens)
    want = ref.attend(q, kc, vc, table, lens, scale, window, exact_scores=exact)
    assert_within(o, want[0], want[2], "o")
    live = lens > 0
    assert_within(lse[live], want[1][live.cpu()], want[3][live.cpu()], "lse")
    assert (lse[~live] == -math.inf).all() and (o[~live] == 0).all()


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("H, Hkv, D", [
    (1, 1, 64), (32, 8, 128), (4, 4, 128), (12, 2, 80), (6, 1, 96), (8, 1, 40), (16, 1, 128),
    (24, 1, 64), (17, 1, 128), (33, 1, 72), (64, 2, 128), (80, 1, 256), (16, 8, 192), (3, 3, 8),
    (20, 1, 104), (40, 1, 96),
])
def test_heads_and_widths(H, Hkv, D, dtype):
    _attend([70, 1, 0, 200], H, Hkv, D, 16, dtype)


@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("P", [1, 2, 7, 16, 64, 100, 256])
@pytest.mark.parametrize("lens", [
    [1], [15], [16], [17], [63], [64], [65], [0, 0, 129, 0], [127, 128, 3], [1000, 5, 64, 0, 333],
])
def test_lengths_and_pages(lens, P, layout):
    _attend(lens, 4, 2, 64, P, torch.bfloat16, layout)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("lens", [
    [5000], [20000], [1, 9000, 17, 0, 4000], [300] * 100, [64] * 400, [1] * 700, list(range(200)),
    [0] * 300 + [777] + [0] * 300,
])
def test_splits(lens, dtype):
    """One item over many CTAs, CTAs of many items, items that begin and end inside a CTA."""
    _attend(lens, 2, 1, 64, 16, dtype)


def test_many_sequences():
    """More than a warp finds its place among in two looks."""
    _attend([3] * 1500 + [70] + [0] * 40 + [130, 1], 1, 1, 64, 16, torch.float16)


@pytest.mark.parametrize("H, Hkv, D, lens", [
    (2, 1, 64, [500, 0, 33]), (32, 32, 128, [200] * 6), (4, 2, 192, [90] * 100), (2, 2, 256, [90] * 100),
])
def test_tables_with_room_to_spare(H, Hkv, D, lens):
    _attend(lens, H, Hkv, D, 16, torch.bfloat16, extra=700)


@pytest.mark.parametrize("H, Hkv, D, count", [
    (12, 6, 80, 30), (12, 12, 40, 16), (8, 8, 128, 90), (8, 8, 64, 90), (32, 1, 96, 200), (3, 3, 192, 60),
    (4, 4, 256, 50),
])
def test_each_size_of_cta(H, Hkv, D, count):
    """Numbers of items on both sides of the rules, whole and shared."""
    lens = [int(n) for n in torch.randint(0, 400, (count,))]
    _attend(lens, H, Hkv, D, 16, torch.float16)
    _attend(lens[:5] + [3000], H, Hkv, D, 16, torch.bfloat16, "head")


@pytest.mark.parametrize("H, Hkv, D", [(8, 8, 128), (40, 2, 128), (32, 1, 256), (16, 4, 192)])
def test_splits_of_many_heads(H, Hkv, D):
    _attend([3000, 1, 700, 0, 64], H, Hkv, D, 32, torch.float16)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 200, 10000])
def test_window(window):
    _attend([0, 1, 64, 65, 500, 1500], 4, 2, 64, 16, torch.bfloat16, window=window)
    _attend([0, 1, 64, 65, 500, 1500], 4, 2, 64, 7, torch.float16, "head", window=window)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("scale", [None, 1.0, 0.0, -0.3])
def test_ordinary_numbers(scale, dtype):
    _attend([300, 7, 1200], 8, 2, 128, 16, dtype, scale=scale, exact=False)


def test_one_key_takes_all():
    """A score far above the others', first, last or between, and far below."""
    D, P, n = 64, 16, 1000
    table, pages = _table([n], P)
    kc, vc = _cache(pages, P, 1, D, torch.float16), _cache(pages, P, 1, D, torch.float16)
    kc.mul_(0.01)
    q = torch.ones(1, 3, D, device="cuda", dtype=torch.float16)
    op = PagedAttentionDecodeOp(3, 1, D, P, dtype=torch.float16)
    for at in (0, 1, 63, 64, 500, n - 1):
        for size in (40.0, -40.0):
            page, slot = int(table[0, at // P]), at % P
            keep = kc[page, slot].clone()
            kc[page, slot] = size
            o, lse = op(q, kc, vc, table, _lens([n]))
            want = ref.attend(q, kc, vc, table, _lens([n]))
            assert_within(o, want[0], want[2], f"o, key {at}")
            assert_within(lse, want[1], want[3], f"lse, key {at}")
            if size > 0:
                assert torch.equal(o[0], vc[page, slot].expand(3, D))
            kc[page, slot] = keep


def test_infinities_and_nan():
    """-inf scores have no weight; +inf and NaN make their head's row NaN and no other's."""
    D, P, n = 64, 16, 300
    table, pages = _table([n, n], P)
    kc, vc = _cache(pages, P, 2, D, torch.bfloat16), _cache(pages, P, 2, D, torch.bfloat16)
    q = torch.rand(2, 4, D, device="cuda").to(torch.bfloat16) + 0.5
    op = PagedAttentionDecodeOp(4, 2, D, P)
    clean, lse0 = op(q, kc, vc, table, _lens([n, n]))
    for at, value in ((10, math.inf), (299, math.nan), (0, math.inf)):
        bad = kc.clone()
        bad[int(table[1, at // P]), at % P, 1] = value
        o, lse = op(q, bad, vc, table, _lens([n, n]))
        assert torch.equal(o[0], clean[0]) and torch.equal(o[1, :2], clean[1, :2])
        assert torch.equal(lse[0], lse0[0]) and torch.equal(lse[1, :2], lse0[1, :2])
        assert o[1, 2:].isnan().all() and lse[1, 2:].isnan().all()
    less = kc.clone()  # every key but the first 5 at -inf: what is left is a sequence of 5
    for at in range(5, n):
        less[int(table[1, at // P]), at % P] = -math.inf
    o, lse = op(q, less, vc, table, _lens([n, n]))
    want = ref.attend(q, kc, vc, table, _lens([n, 5]))
    assert_within(o, want[0], want[2])
    assert_within(lse, want[1], want[3])
    for at in range(5):
        less[int(table[1, at // P]), at % P] = -math.inf
    o, lse = op(q, less, vc, table, _lens([n, n]))  # no key with a weight
    assert (o[1] == 0).all() and (lse[1] == -math.inf).all() and torch.equal(o[0], clean[0])


def test_fp16_keeps_small_weights():
    """One weight of 1 and thousands of 2^-20, which fp16 alone would hold in 4 bits."""
    D, P, n = 64, 16, 8000
    table, pages = _table([n], P)
    kc = _cache(pages, P, 1, D, torch.float16, fill=0.0)
    vc = _cache(pages, P, 1, D, torch.float16, fill=1.0)
    at = 77
    kc[int(table[0, at // P]), at % P, 0, 0] = 20.3
    vc[int(table[0, at // P]), at % P] = 0.0
    q = torch.zeros(1, 1, D, device="cuda", dtype=torch.float16)
    q[0, 0, 0] = 1.0
    op = PagedAttentionDecodeOp(1, 1, D, P, math.log(2.0), dtype=torch.float16)
    o, _ = op(q, kc, vc, table, _lens([n]))
    want = 1.0 / (1.0 + 2.0 ** float(kc[int(table[0, 4]), 13, 0, 0]) / (n - 1))
    # The weights all round alike, half a step, and so does the output; the rest is below 2^-14.
    assert abs(float(o[0, 0, 0]) - want) < want * (2**-10 + 2**-14)


def test_shared_prefix_pages_and_a_cache_without_pages():
    D, P = 64, 16
    kc, vc = _cache(9, P, 2, D, torch.bfloat16), _cache(9, P, 2, D, torch.bfloat16)
    table = torch.tensor([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 2, 6]], dtype=torch.int32, device="cuda")
    q = torch.randn(3, 4, D, device="cuda").to(torch.bfloat16)
    o, lse = PagedAttentionDecodeOp(4, 2, D, P)(q, kc, vc, table, _lens([60, 64, 49]))
    want = ref.attend(q, kc, vc, table, _lens([60, 64, 49]))
    assert_within(o, want[0], want[2])
    assert_within(lse, want[1], want[3])
    k, v = (torch.randn(3, 200, 2, D, device="cuda").to(torch.bfloat16) for _ in range(2))
    table = torch.arange(3, dtype=torch.int32, device="cuda")[:, None]
    o, lse = PagedAttentionDecodeOp(4, 2, D, 200)(q, k, v, table, _lens([200, 3, 77]))
    want = ref.attend(q, k, v, table, _lens([200, 3, 77]))
    assert_within(o, want[0], want[2])


def test_layouts():
    """q as a column slice, keys and values side by side in one buffer, a table with wide rows."""
    D, P, lens = 64, 16, [100, 33, 0]
    table, pages = _table(lens, P)
    wide = torch.full((3, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + table.shape[1]] = table
    both = torch.randn(pages, P, 2, 2, D, device="cuda").to(torch.bfloat16)
    kc, vc = both[:, :, 0], both[:, :, 1]
    qkv = torch.randn(3, 4 * D + 24, device="cuda").to(torch.bfloat16)
    op = PagedAttentionDecodeOp(4, 2, D, P)
    for q in (qkv[:, 24:], qkv[:, 3:3 + 4 * D], torch.randn(D, 4, 3, device="cuda").bfloat16().permute(2, 1, 0).flip(2)):
        q = q.unflatten(1, (4, D)) if q.dim() == 2 else q
        for t in (table, wide[:, 5:], table.t().contiguous().t()):
            o, lse = op(q, kc, vc, t, _lens(lens))
            want = ref.attend(q, kc, vc, t, _lens(lens))
            assert_within(o, want[0], want[2])
            assert_within(lse[:2], want[1][:2], want[3][:2])
    spread = torch.tensor([100, 9, 33, 9, 0, 9], dtype=torch.int32, device="cuda")[::2]
    assert torch.equal(op(q, kc, vc, table, spread)[0], o)


def test_nothing_to_do():
    kc = _cache(1, 16, 2, 64, torch.bfloat16)
    op = PagedAttentionDecodeOp(4, 2, 64, 16)
    o, lse = op(torch.empty(0, 4, 64, device="cuda", dtype=torch.bfloat16), kc, kc,
                torch.empty(0, 3, dtype=torch.int32, device="cuda"), _lens([]))
    assert o.shape == (0, 4, 64) and lse.shape == (0, 4)
    q = torch.randn(2, 4, 64, device="cuda").to(torch.bfloat16)
    o, lse = op(q, kc, kc, torch.empty(2, 0, dtype=torch.int32, device="cuda"), _lens([0, -5]))
    assert (o == 0).all() and (lse == -math.inf).all()


def test_repeats_to_the_bit_and_runs_on_two_streams():
    lens = [4000, 17, 900, 0, 2500]
    table, pages = _table(lens, 16)
    kc, vc = _cache(pages, 16, 2, 128, torch.bfloat16), _cache(pages, 16, 2, 128, torch.bfloat16)
    q = torch.randn(5, 8, 128, device="cuda").to(torch.bfloat16)
    op = PagedAttentionDecodeOp(8, 2, 128, 16)
    want = op(q, kc, vc, table, _lens(lens))
    lens = _lens(lens)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for s in side:
            with torch.cuda.stream(s):
                got.append(op(q, kc, vc, table, lens))
    torch.cuda.synchronize()
    for o, lse in got:
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_a_kept_workspace_serves_calls_of_all_kinds():
    """Calls of several sizes on one stream, each of which shares items among CTAs, from two host
    threads and on two streams at once; the counters are zero behind them."""
    import threading

    from tileops.kernels.attention import paged_attention as kernels

    made = []
    for lens, H, Hkv, D in (([3000], 2, 1, 64), ([900, 5000, 0, 77], 16, 2, 128), ([2000] * 3, 4, 4, 192),
                            ([4000, 4000], 40, 1, 96)):
        table, pages = _table(lens, 16)
        kc, vc = _cache(pages, 16, Hkv, D, torch.bfloat16), _cache(pages, 16, Hkv, D, torch.bfloat16)
        q = torch.randn(len(lens), H, D, device="cuda").to(torch.bfloat16)
        args = (q, kc, vc, table, _lens(lens))
        made.append((PagedAttentionDecodeOp(H, Hkv, D, 16), args, ref.attend(*args)))
    want = [op(*args) for op, args, _ in made]
    for (o, lse), (_, _, exact) in zip(want, made):
        assert_within(o, exact[0], exact[2])
    wrong = []

    def work(stream):
        with torch.cuda.stream(stream):
            for _ in range(30):
                for (op, args, _), (o, lse) in zip(made, want):
                    got = op(*args)
                    if not (torch.equal(got[0], o) and torch.equal(got[1].nan_to_num(neginf=0.0),
                                                                   lse.nan_to_num(neginf=0.0))):
                        wrong.append(args[0].shape)

    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    threads = [threading.Thread(target=work, args=(s,)) for s in (streams[0], streams[0], streams[1])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not wrong
    for ws in kernels._workspaces.values():
        assert not ws[:4 * 592].any()


def test_a_graph_and_calls_beside_it():
    """A captured step has a workspace of its own: replayed on one stream while calls run on another."""
    lens = _lens([4000, 100])
    table, pages = _table([4000, 100], 16)
    kc, vc = _cache(pages, 16, 1, 64, torch.bfloat16), _cache(pages, 16, 1, 64, torch.bfloat16)
    q = torch.randn(2, 2, 64, device="cuda").to(torch.bfloat16)
    op = PagedAttentionDecodeOp(2, 1, 64, 16)
    want = op(q, kc, vc, table, lens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = op(q, kc, vc, table, lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(50):
        graph.replay()
        with torch.cuda.stream(side):
            beside = op(q, kc, vc, table, lens)
    torch.cuda.synchronize()
    for o, lse in (got, beside):
        assert torch.equal(o, want[0]) and torch.equal(lse, want[1])


def test_two_graphs_of_one_pool():
    """Two captured steps that may share their workspace's memory, replayed in turn with lengths
    that change between replays."""
    lens = _lens([300, 0, 2000])
    table, pages = _table([2100, 2100, 2100], 16)
    kc, vc = _cache(pages, 16, 1, 64, torch.bfloat16), _cache(pages, 16, 1, 64, torch.bfloat16)
    q = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    op = PagedAttentionDecodeOp(2, 1, 64, 16)
    op(q, kc, vc, table, lens)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    pool = torch.cuda.graph_pool_handle()
    for g in graphs:
        with torch.cuda.graph(g, pool=pool):
            outs.append(op(q, kc, vc, table, lens))
    for now in ([300, 0, 2000], [1, 2100, 64], [0, 0, 0], [2100, 2100, 2100]):
        lens.copy_(torch.tensor(now, dtype=torch.int32))
        for g in graphs:
            g.replay()
        want = ref.attend(q, kc, vc, table, lens)
        for o, lse in outs:
            assert_within(o, want[0], want[2], str(now))
            live = lens > 0
            assert_within(lse[live], want[1][live.cpu()], want[3][live.cpu()])


def test_a_first_call_inside_a_capture():
    """An op's first call of its kind captured (another has looked the device's error flag up)."""
    table, pages = _table([70, 200], 16)
    lens = _lens([70, 200])
    kc, vc = _cache(pages, 16, 3, 72, torch.bfloat16), _cache(pages, 16, 3, 72, torch.bfloat16)
    q, k = (torch.randn(2, n, 72, device="cuda").to(torch.bfloat16) for n in (6, 3))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        qr = PagedKVAppendOp(3, 72, 16, 6, 20, True)(k, k, kc, vc, table, lens, q)
        o, lse = PagedAttentionDecodeOp(6, 3, 72, 16, window=100)(qr, kc, vc, table, lens)
    expect = ref.append(k, k, kc, vc, table, lens, rotary_frequencies(20), q, interleaved=True)
    graph.replay()
    assert_within(qr, expect[0], expect[1])
    assert_within(kc, expect[2], expect[3])
    want = ref.attend(qr, kc, vc, table, lens, window=100)
    assert_within(o, want[0], want[2])
    assert_within(lse, want[1], want[3])


def test_offsets_past_32_bits():
    """Pages more than 2^32 elements apart."""
    far = torch.empty(2**32 + 2**16, dtype=torch.bfloat16, device="cuda")
    kc = far.as_strided((2, 16, 2, 64), (2**32, 128, 64, 1))
    vc = far.as_strided((2, 16, 2, 64), (2**32, 128, 64, 1), 4096)
    kc.normal_()
    vc.normal_()
    table = torch.tensor([[1, 0]], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 4, 64, device="cuda").to(torch.bfloat16)
    o, lse = PagedAttentionDecodeOp(4, 2, 64, 16)(q, kc, vc, table, _lens([30]))
    want = ref.attend(q, kc, vc, table, _lens([30]))
    assert_within(o, want[0], want[2])
    k, v = (torch.randn(1, 30, 2, 64, device="cuda").to(torch.bfloat16) for _ in range(2))
    PagedKVAppendOp(2, 64, 16)(k, v, kc, vc, table, _lens([30]))
    assert torch.equal(kc[1], k[0, :16]) and torch.equal(kc[0, :14], k[0, 16:])
    assert torch.equal(vc[1], v[0, :16]) and torch.equal(vc[0, :14], v[0, 16:])


def test_a_token_without_a_page_sets_the_flag():
    kc, vc = _cache(4, 16, 1, 64, torch.bfloat16), _cache(4, 16, 1, 64, torch.bfloat16)
    q = torch.randn(1, 1, 64, device="cuda").to(torch.bfloat16)
    op = PagedAttentionDecodeOp(1, 1, 64, 16)
    for table, n in (([0, 4], 20), ([0, -1], 20), ([1, 2], 33), ([1, 2], 2**31 - 1)):
        table = torch.tensor([table], dtype=torch.int32, device="cuda")
        op(q, kc, vc, table, _lens([n]))
        assert _flag() == 3
    op(q, kc, vc, torch.tensor([[0, 99]], dtype=torch.int32, device="cuda"), _lens([16]))
    assert _flag() == 0  # the entry is of no token in use


# ------------------------------------------------------------ append
def _append(lens, new, H, Hkv, D, P, dtype, layout="token", packed=False, R=None, interleaved=False,
            frequencies=None, amplitude=1.0, tail=0, queries=True, extra=0):
    R = D if R is None else R
    f = rotary_frequencies(R) if frequencies is None else frequencies
    table, pages = _table(lens, P, extra)
    kc, vc = _cache(pages, P, Hkv, D, dtype, layout), _cache(pages, P, Hkv, D, dtype, layout)
    cu = None
    if packed:
        cu = torch.tensor([0, *new]).cumsum(0).to(torch.int32).cuda()
        rows = (sum(new) + tail,)
    else:
        rows = (len(lens),) if new == 1 else (len(lens), new)
    q, k, v = (torch.randn(*rows, h, D, device="cuda").to(dtype) for h in (H, Hkv, Hkv))
    q = q if queries else None
    want = ref.append(k, v, kc, vc, table, _lens(lens), f, q, cu, amplitude, interleaved)
    op = PagedKVAppendOp(Hkv, D, P, H, R, interleaved, frequencies, amplitude, dtype)
    got = op(k, v, kc, vc, table, _lens(lens), q, cu)
    if queries:
        assert_within(got, want[0], want[1], "q")
    else:
        assert got is None
    assert_within(kc, want[2], want[3], "k_cache")
    assert torch.equal(vc.cpu().double(), want[4])
    live = (want[3] > 0).any(-1)  # slots that nothing was written to are as they were
    assert_within(kc[~live], want[2][~live], torch.zeros_like(want[2][~live]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("layout", ["token", "head"])
@pytest.mark.parametrize("P", [1, 7, 16, 64])
@pytest.mark.parametrize("lens, new", [
    ([1], 1), ([100], 1), ([5, 0, 64, 17], 1), ([40], 40), ([40, 16, 0], 7), ([3, 2, 50], 5),
])
def test_append(lens, new, P, layout, dtype):
    _append(lens, new, 4, 2, 64, P, dtype, layout)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new", [
    ([9], [9]), ([20, 64, 5], [4, 64, 1]), ([0, 30, 30, 7], [0, 0, 30, 2]), ([5, 3], [9, 9]),
    ([100] * 40, [1, 2, 3, 0] * 10),
])
@pytest.mark.parametrize("tail", [0, 5])
def test_append_packed(lens, new, tail, dtype):
    _append(lens, new, 4, 1, 64, 16, dtype, packed=True, tail=tail)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H, Hkv, D, R, interleaved", [
    (1, 1, 8, 0, False), (32, 8, 128, 128, False), (3, 1, 80, 40, True), (2, 2, 33, 10, False),
    (2, 2, 33, 10, True), (5, 1, 256, 256, True), (2, 1, 50, 50, False), (64, 4, 96, 96, False),
])
def test_append_heads_and_rotations(H, Hkv, D, R, interleaved, dtype):
    _append([50, 3, 77], 3, H, Hkv, D, 16, dtype, R=R, interleaved=interleaved)
    _append([50, 3, 77], [3, 3, 20], H, Hkv, D, 16, dtype, packed=True, R=R,
            interleaved=interleaved, queries=False)


def test_append_scaled():
    f = rotary_frequencies(64, factor=8.0, original_length=4096)
    _append([5000, 12], 12, 2, 1, 64, 32, torch.float32, frequencies=f, amplitude=1.2)


def test_append_many_tokens():
    _append([700, 2000], [700, 1500], 3, 1, 64, 16, torch.bfloat16, packed=True, tail=100)


def test_append_layouts():
    """Slices of one projection's output, keys and values in one buffer."""
    D, P, lens = 64, 16, [40, 7]
    table, pages = _table(lens, P)
    both = torch.randn(pages, P, 2, 2, D, device="cuda")
    keep = both.clone()
    qkv = torch.randn(2, 5, 8 * D, device="cuda")
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([4 * D, 2 * D, 2 * D], dim=-1))
    want = ref.append(k, v, keep[:, :, 0], keep[:, :, 1], table, _lens(lens), rotary_frequencies(D), q)
    got = PagedKVAppendOp(2, D, P, 4, D, dtype=torch.float32)(
        k, v, both[:, :, 0], both[:, :, 1], table, _lens(lens), q)
    assert_within(got, want[0], want[1])
    assert_within(both[:, :, 0], want[2], want[3])
    assert torch.equal(both[:, :, 1].cpu().double(), want[4])


def test_append_nothing():
    kc, vc = _cache(2, 16, 1, 64, torch.bfloat16), _cache(2, 16, 1, 64, torch.bfloat16)
    keep = kc.clone(), vc.clone()
    op = PagedKVAppendOp(1, 64, 16, 2, 64)
    none = torch.empty(0, 1, 64, device="cuda", dtype=torch.bfloat16)
    q = torch.empty(0, 2, 64, device="cuda", dtype=torch.bfloat16)
    table = torch.zeros(0, 1, dtype=torch.int32, device="cuda")
    assert op(none, none, kc, vc, table, _lens([]), q).shape == (0, 2, 64)
    row = torch.randn(3, 1, 64, device="cuda").to(torch.bfloat16)
    q = torch.randn(3, 2, 64, device="cuda").to(torch.bfloat16)
    got = op(row, row, kc, vc, table, _lens([]), q, torch.zeros(1, dtype=torch.int32, device="cuda"))
    assert (got == 0).all()  # rows behind the last sequence
    assert torch.equal(kc, keep[0]) and torch.equal(vc, keep[1])


def test_append_refused_on_the_device_sets_the_flag():
    """Nothing but the good tokens is written."""
    kc, vc = _cache(4, 16, 1, 64, torch.float32), _cache(4, 16, 1, 64, torch.float32)
    op = PagedKVAppendOp(1, 64, 16, dtype=torch.float32)
    k, v = torch.randn(1, 20, 1, 64, device="cuda"), torch.randn(1, 20, 1, 64, device="cuda")
    for table, n in (([0, 4], 20), ([0, -1], 20), ([0], 20)):
        keep = kc.clone()
        op(k, v, kc, vc, torch.tensor([table], dtype=torch.int32, device="cuda"), _lens([n]))
        assert _flag() == 3
        assert torch.equal(kc[0], k[0, :16]) and torch.equal(kc[1:], keep[1:])
    op(k, v, kc, vc, torch.tensor([[0, 1]], dtype=torch.int32, device="cuda"), _lens([2**31 - 1]))
    assert _flag() == 3
    k, v = k[0], v[0]
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device="cuda")
    for cu in ([0, 15, 10], [3, 5, 20], [0, 5, 21], [0, 2**31 - 1, -(2**31)]):
        op(k, v, kc, vc, table, _lens([20, 20]), None, torch.tensor(cu, dtype=torch.int32, device="cuda"))
        assert _flag() in (2, 3)


# ------------------------------------------------------------ scores of any size
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("scale", [1e3, 1e4, 1e6, -1e6, 1e8, 2.0**100])
@pytest.mark.parametrize("n", [30, 1000, 30000])
def test_scores_of_any_size(n, scale, dtype):
    """A weight is relative to the largest score's, whose own is 1 whatever the scale: a key far above
    the others takes all, wherever it lies among warps and CTAs, and two such keys half each."""
    D, P = 64, 16
    table, pages = _table([n], P)
    kc, vc = _cache(pages, P, 1, D, dtype), _cache(pages, P, 1, D, dtype)
    kc.mul_(0.01)
    q = torch.ones(1, 3, D, device="cuda", dtype=dtype)
    op = PagedAttentionDecodeOp(3, 1, D, P, scale, dtype=dtype)

    def slot(at):
        return int(table[0, at // P]), at % P

    for size in (40.0, 38.75, 12.125):  # sums of 64 of them are exact in both types
        size = math.copysign(size, scale)
        for first, second in ((0, n - 1), (n // 2, 3), (n - 1, n // 3)):
            kept = kc.clone()
            top = abs(64 * size * scale) / math.log(2.0)
            kc[slot(first)] = size
            o, lse = op(q, kc, vc, table, _lens([n]))
            assert torch.equal(o[0], vc[slot(first)].expand(3, D)), (size, first)
            # log2(e) scale, its product with the score and the sum round once each
            assert ((lse.double() - top).abs() <= 4 * ref.U * top).all(), (size, first, lse)
            kc[slot(second)] = size
            o, lse = op(q, kc, vc, table, _lens([n]))
            a, b = (vc[slot(at)].double().expand(3, D).cpu() for at in (first, second))
            # the sum may cut (2 u of its terms), its product with 1 / 2 rounds
            assert_within(o[0], (a + b) / 2, 4 * ref.U * (a.abs() + b.abs()))
            assert ((lse.double() - (top + 1)).abs() <= 4 * ref.U * (top + 1)).all(), (size, second, lse)
            kc.copy_(kept)


# ------------------------------------------------------------ the longest sequences
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("window", [None, 300, 2**30])
@pytest.mark.parametrize("P, columns", [(2**31 - 129, 1), (21474835, 100), (17043519, 126)])
def test_the_longest_sequences(P, columns, window, dtype):
    """As many tokens as a table may have room for, in pages whose slots all lie in one place: units
    of 256 tokens end beyond 2^31.  The values of the first pages are 1, of the last tenth 3; all
    keys are alike."""
    D, room = 8, P * columns
    assert 2**31 - 255 <= room <= 2**31 - 129
    kc = torch.ones(2, 1, 1, D, device="cuda", dtype=dtype).expand(2, P, 1, D)
    vc = (kc[:, :1] * torch.tensor([1.0, 3.0], device="cuda", dtype=dtype)[:, None, None, None]).expand(2, P, 1, D)
    first = columns - columns // 10  # page of the first 3
    table = (torch.arange(columns, device="cuda")[None] >= first).to(torch.int32)
    q = torch.ones(1, 1, D, device="cuda", dtype=dtype)
    op = PagedAttentionDecodeOp(1, 1, D, P, 0.25, window, dtype)
    for n in (room, room - 1, room - 254) if window == 300 else (room,):
        o, lse = op(q, kc, vc, table, _lens([n]))
        seen = min(n, window or n)
        threes = min(seen, max(0, n - first * P))
        want = torch.full((1, 1, D), 1.0 + 2.0 * threes / seen, dtype=torch.float64)
        # A warp's sums are whole numbers below 2^24; those of 8 warps and up to 148 CTAs round.
        assert_within(o, want, 64 * ref.U * want, f"o, {n} tokens")
        want = math.log2(seen) + 2.0 / math.log(2.0)
        assert abs(float(lse) - want) <= 8 * ref.U * want + 64 * ref.U, (n, float(lse), want)
    if window:
        got = op(q, kc, vc, table, _lens([2**31 - 1]))  # longer than the table: taken as its room
        assert _flag() == 3
        for a, b in zip(got, op(q, kc, vc, table, _lens([room]))):
            assert torch.equal(a, b)


# ------------------------------------------------------------ streams
def test_streams_that_are_not_torchs():
    """An external stream's calls keep nothing; the per-thread default stream, one handle and a stream
    in each thread, serves threads at once; torch's own streams are told apart by their numbers."""
    from concurrent.futures import ThreadPoolExecutor

    from tileops.kernels.attention import paged_attention as kernels

    own = torch.cuda.Stream()
    assert own.stream_id % 2 == 1 and torch.cuda.default_stream().stream_id == 0
    external = torch.cuda.ExternalStream(own.cuda_stream)
    assert external.stream_id == own.cuda_stream and external.stream_id % 2 == 0
    made = []
    for lens, H, Hkv, D in (([3000, 20], 2, 1, 64), ([900, 5000, 0, 77], 16, 2, 128), ([9000], 40, 1, 96)):
        table, pages = _table(lens, 16)
        kc, vc = _cache(pages, 16, Hkv, D, torch.bfloat16), _cache(pages, 16, Hkv, D, torch.bfloat16)
        q = torch.randn(len(lens), H, D, device="cuda").to(torch.bfloat16)
        args = (q, kc, vc, table, _lens(lens))
        op = PagedAttentionDecodeOp(H, Hkv, D, 16)
        made.append((op, args, op(*args)))
    torch.cuda.synchronize()
    kept = dict(kernels._workspaces)

    def work(handle):
        with torch.cuda.stream(torch.cuda.ExternalStream(handle)):
            return [(n, op(*args)) for _ in range(40) for n, (op, args, _) in enumerate(made)]

    per_thread = 2
    with ThreadPoolExecutor(3) as pool:
        runs = [pool.submit(work, h) for h in (per_thread, per_thread, per_thread, own.cuda_stream)]
        got = [r.result() for r in runs]
        torch.cuda.synchronize()
    for calls in got:
        assert len(calls) == 40 * len(made)
        for n, (o, lse) in calls:
            assert torch.equal(o, made[n][2][0]) and torch.equal(lse, made[n][2][1])
    assert kernels._workspaces.keys() == kept.keys()


# ------------------------------------------------------------ small scales
@pytest.mark.parametrize("scale", [0.0, 1e-33, -1e-33, 3e-32, 1e-31, 1e-44])
def test_small_scales_of_large_scores(scale):
    """Scores of 2^100 and more (their sums are exact) under a scale that brings them near zero, or
    to nothing: all tokens count alike then."""
    D, P, lens = 64, 16, [40, 700]
    table, pages = _table(lens, P)
    kc = _whole(pages, P, 2, D, dtype=torch.bfloat16) * 2.0**50
    vc = _cache(pages, P, 2, D, torch.bfloat16)
    q = _whole(2, 4, D, dtype=torch.bfloat16) * 2.0**50
    o, lse = PagedAttentionDecodeOp(4, 2, D, P, scale)(q, kc, vc, table, _lens(lens))
    want = ref.attend(q, kc, vc, table, _lens(lens), scale, exact_scores=True)
    assert_within(o, want[0], want[2], "o")
    assert_within(lse, want[1], want[3], "lse")


def test_threads_and_streams_finish_all_their_calls():
    """Two host threads on one of torch's streams and one on another: every call's result is counted
    and compared; a thread that raises fails the test."""
    from concurrent.futures import ThreadPoolExecutor

    made = []
    for lens, H, Hkv, D in (([3000], 2, 1, 64), ([900, 5000, 0, 77], 16, 2, 128), ([2000] * 3, 4, 4, 192),
                            ([4000, 4000], 40, 1, 96)):
        table, pages = _table(lens, 16)
        kc, vc = _cache(pages, 16, Hkv, D, torch.bfloat16), _cache(pages, 16, Hkv, D, torch.bfloat16)
        q = torch.randn(len(lens), H, D, device="cuda").to(torch.bfloat16)
        args = (q, kc, vc, table, _lens(lens))
        op = PagedAttentionDecodeOp(H, Hkv, D, 16)
        made.append((op, args, op(*args)))
    torch.cuda.synchronize()

    def work(stream):
        done = 0
        with torch.cuda.stream(stream):
            for _ in range(30):
                for op, args, (o, lse) in made:
                    got = op(*args)
                    assert torch.equal(got[0], o) and torch.equal(got[1], lse)
                    done += 1
        return done

    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    with ThreadPoolExecutor(3) as pool:
        runs = [pool.submit(work, s) for s in (streams[0], streams[0], streams[1])]
        assert [r.result() for r in runs] == [30 * len(made)] * 3
    torch.cuda.synchronize()


# ------------------------------------------------------------ what weights are held in
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("H, Hkv", [(1, 1), (8, 1), (16, 2), (21, 3), (4, 4)])
@pytest.mark.parametrize("D", [64, 96, 128, 192, 256])
def test_weights_of_up_to_8_heads_keep_more_bits_than_the_type(D, H, Hkv, dtype):
    """Half of the tokens have the value 1, half -1, and scores that differ little: what is left of o
    after the cancellation are the weights' differences, which their type alone does not hold."""
    P, n = 16, 64
    table, pages = _table([n], P)
    kc = _cache(pages, P, Hkv, D, dtype, fill=0.0)
    vc = _cache(pages, P, Hkv, D, dtype, fill=1.0)
    q = torch.zeros(1, H, D, device="cuda", dtype=dtype)
    q[..., 5] = 1.0
    odd = torch.randperm(n, device="cuda")[:n // 2]
    at = table[0].long()[odd // P], odd % P
    vc[at] = -1.0
    op = PagedAttentionDecodeOp(H, Hkv, D, P, math.log(2.0), dtype=dtype)  # scores are exponents of 2
    for less in (2.0**-10, 3 * 2.0**-9, 0.3, 2.7):
        kc[at + (slice(None), 5)] = -less
        w = 2.0 ** -float(torch.tensor(less, dtype=dtype))
        o, _ = op(q, kc, vc, table, _lens([n]))
        half = torch.finfo(dtype).eps / 2
        # each weight half a step of half a step off, 8 u of its exponential, sums of n terms 2 u each
        bound = half**2 + 8 * ref.U + 2 * ref.U * (n + 64)
        want = torch.full((1, H, D), (1 - w) / (1 + w), dtype=torch.float64)
        assert_within(o, want, torch.full_like(want, bound), f"{less}")


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("H, Hkv", [(1, 1), (8, 1), (9, 1), (32, 1), (4, 2)])
@pytest.mark.parametrize("n", [5, 3000])
def test_infinite_values(n, H, Hkv, dtype):
    """An infinite value makes its channel infinite, whatever its weight's bits are; two that differ in
    sign, and NaN, make it NaN; no other channel is touched."""
    D, P = 64, 16
    table, pages = _table([n], P)
    kc, vc = _cache(pages, P, Hkv, D, dtype, fill=0.0), _cache(pages, P, Hkv, D, dtype)
    kc[..., 0] = (torch.rand(pages, P, Hkv, device="cuda") * -3).to(dtype)
    kc[int(table[0, 0]), 0, :, 0] = 1.0  # the largest weight is a whole one
    q = torch.zeros(1, H, D, device="cuda", dtype=dtype)
    q[..., 0] = 1.0
    op = PagedAttentionDecodeOp(H, Hkv, D, P, 1.0, dtype=dtype)
    clean, _ = op(q, kc, vc, table, _lens([n]))
    for channel, at in ((3, 0), (17, 1), (40, n - 1)):
        vc[int(table[0, at // P]), at % P, :, channel] = math.inf
    vc[int(table[0, 0]), 2, :, 8] = -math.inf
    vc[int(table[0, 0]), 1, :, 9] = math.inf
    vc[int(table[0, 0]), 3, :, 9] = -math.inf
    vc[int(table[0, 0]), 4, :, 10] = math.nan
    o, _ = op(q, kc, vc, table, _lens([n]))
    assert (o[..., [3, 17, 40]] == math.inf).all() and (o[..., 8] == -math.inf).all()
    assert o[..., [9, 10]].isnan().all()
    rest = [c for c in range(D) if c not in (3, 17, 40, 8, 9, 10)]
    assert torch.equal(o[..., rest], clean[..., rest])
