"""The operators between the packed linears through the C ABI, against plain implementations in 64 bits: the norms around a block, the
paged 8-bit cache, the attention over it, the upkeep of its pages; and what they refuse."""
import math
import os
import random

import pytest

import __graft_entry__ as entry

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
BLOCK = 16


@pytest.fixture(scope="module")
def qi():
    if not torch.cuda.is_available():
        pytest.fail("the gpu tests need a CUDA device")
    module = entry.load_package()
    if not os.path.exists(module.LIB_PATH):
        module.build()
    module.lib()
    return module


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def settled(qi):
    torch.cuda.synchronize()
    assert qi.kernel_status() == 0


class Store:
    """A pool with sequences in scattered pages, and the values that it holds in 64 bits."""

    def __init__(self, qi, seed, lengths, *, kv_heads=2, head_dim=128, page=32, layers=2, layer=1, spare=3, table_extra=0, fill=True):
        self.qi, self.layer, self.page, self.kv_heads, self.head_dim, self.lengths_list = qi, layer, page, kv_heads, head_dim, lengths
        rng = random.Random(seed)
        needed = [-(-n // page) for n in lengths]
        pages = max(sum(needed) + spare, 1)
        order = list(range(pages))
        rng.shuffle(order)
        width = max(needed + [1]) + table_extra
        references, table = [0] * pages, []
        for n in needed:
            mine = [order.pop() for _ in range(n)]
            for p in mine:
                references[p] = 1
            table.append(mine + [-1] * (width - n))
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape, scales = (layers, pages, kv_heads, page, head_dim), (layers, pages, kv_heads, page // BLOCK)
        self.codes, self.scales = {}, {}
        for which in "kv":
            if fill:
                self.codes[which] = (torch.randn(*shape, device="cuda", generator=g) * 40 + 128).round().clamp(1, 255).to(torch.uint8)
                self.scales[which] = torch.rand(*scales, device="cuda", generator=g) * 0.03 + 0.01
            else:  # what a fresh allocation may hold
                self.codes[which] = torch.randint(0, 256, shape, device="cuda", generator=g, dtype=torch.uint8)
                self.scales[which] = torch.full(scales, float("nan"), device="cuda")
        self.table, self.lengths, self.references = ints(table), ints(lengths), ints(references)
        if fill:  # nothing may depend on scales of blocks that hold no token
            for s, n in enumerate(lengths):
                for block in range(-(-n // BLOCK), needed[s] * (page // BLOCK)):
                    for which in "kv":
                        self.scales[which][:, table[s][block * BLOCK // page], :, block % (page // BLOCK)] = float("nan")
        self.cache = qi.KvCache(self.codes["k"], self.codes["v"], self.scales["k"], self.scales["v"])
        self.pages = qi.KvPages(self.table, self.lengths, self.references)

    def values(self, which, s, length=None):
        """[tokens, kv_heads, head_dim] in 64 bits."""
        length = self.lengths_list[s] if length is None else length
        mine = self.table[s, : -(-length // self.page)].long()
        codes = self.codes[which][self.layer, mine].transpose(1, 2).reshape(-1, self.kv_heads, self.head_dim)[:length].double() - 128
        scales = self.scales[which][self.layer, mine].transpose(1, 2).reshape(-1, self.kv_heads)
        return codes * scales.double().repeat_interleave(BLOCK, 0)[:length, :, None]

    def batch(self, slots, counts, spare_tokens=0, most=None):
        offsets = [sum(counts[:b]) for b in range(len(counts) + 1)]
        return self.qi.KvBatch(ints(slots), ints(offsets), sum(counts) + spare_tokens, max(counts + [0]) if most is None else most)


# ---- attention ---------------------------------------------------------------------------------------------------
#
# Tolerance. Codes, queries and products are exact; sums are float32. Weights p are rounded to float16 (relative 2^-11 at most, each by
# itself), y to float16 (2^-11). An element of y is a weighted mean of values: |error| <= 2^-11 * sum p|v| / sum p + 2^-11 |y| + the float32
# sums' part, which for 8192 terms in any order is below 2^-13 of the same mean. sum p|v| / sum p <= max |v|, so 2^-10 * max|v| bounds
# every element, and the 2-norm, where the roundings are independent, is below 2^-11 of the result's. lse: 2^-21 * (|lse| + |x| max), x the
# scores in base 2 (the fused multiply-add and ex2.approx, 2^-22 each), below 1e-5 absolute for scores below 16.


def attend_exact(store, q, slots, counts, heads, scale, causal, window):
    ys, lses, begin = [], [], 0
    group = heads // store.kv_heads
    for s, count in zip(slots, counts):
        length = store.lengths_list[s]
        k, v = (store.values(which, s).repeat_interleave(group, 1) for which in "kv")
        mine = q[begin:begin + count].double()
        begin += count
        scores = torch.einsum("ihd,jhd->hij", mine, k) * scale
        p, j = torch.arange(length - count, length, device="cuda")[:, None], torch.arange(length, device="cuda")[None]
        hidden = torch.zeros(count, length, dtype=torch.bool, device="cuda")
        if causal:
            hidden |= j > p
        if window:
            hidden |= j <= p - window
        scores = scores.masked_fill(hidden, -math.inf)
        lse = torch.logsumexp(scores, 2) if length else torch.full((heads, count), -math.inf, dtype=torch.float64, device="cuda")
        weights = torch.exp(scores - torch.where(lse == -math.inf, 0.0, lse)[..., None])
        ys.append(torch.einsum("hij,jhd->ihd", weights, v))
        lses.append(lse.T)
    return torch.cat(ys), torch.cat(lses)


def attend(qi, store, slots, counts, heads, *, causal=True, window=0, seed=1, gap=0, max_length=None, most=None, stream=None, q=None):
    tokens, dim = sum(counts), store.head_dim
    g = torch.Generator(device="cuda").manual_seed(seed)
    if q is None:
        q = (torch.randn(tokens, heads, dim, device="cuda", generator=g) * 1.5).half()
    rows = torch.full((tokens, heads * dim + gap), float("nan"), dtype=torch.float16, device="cuda")
    rows[:, : heads * dim] = q.view(tokens, -1)
    y = torch.full((tokens, heads * dim + gap), float("nan"), dtype=torch.float16, device="cuda")
    lse = torch.full((tokens, heads), float("nan"), device="cuda")
    batch = store.batch(slots, counts, most=most)
    max_length = max(store.lengths_list) if max_length is None else max_length
    workspace = torch.zeros(qi.kv_attention_workspace(store.cache, batch, heads, max_length), dtype=torch.uint8, device="cuda")
    results = []
    for _ in range(2):  # the second call finds the workspace as the first one left it
        if stream is not None:
            stream.wait_stream(torch.cuda.current_stream())
        status = qi.kv_attention_ex(store.cache, store.pages, batch, store.layer, rows, heads * dim + gap, y, heads * dim + gap, heads, dim ** -0.5, max_length, causal=causal,
                                    window=window, lse=lse, workspace=workspace, stream=None if stream is None else stream.cuda_stream)
        assert status == 0
        settled(qi)
        results.append((y.clone(), lse.clone()))
    assert torch.equal(results[0][0].view(torch.int16), results[1][0].view(torch.int16)) and torch.equal(results[0][1], results[1][1]), "two calls, two results"
    assert gap == 0 or y[:, heads * dim:].isnan().all(), "written beyond the row"
    got, exact, exact_lse = y[:, : heads * dim].view(tokens, heads, dim).double(), *attend_exact(store, q, slots, counts, heads, dim ** -0.5, causal, window)
    assert torch.equal(lse == -math.inf, exact_lse == -math.inf)
    seen = exact_lse > -math.inf
    assert (got[~seen] == 0).all()
    if seen.any():
        largest = max(store.values("v", s).abs().max().item() for s in slots if store.lengths_list[s])
        assert not got.isnan().any()
        assert (got - exact).abs().max().item() <= 2.0 ** -10 * largest
        assert (got - exact).norm().item() <= 2.0 ** -11 * exact.norm().item()
        assert (lse.double() - exact_lse)[seen].abs().max().item() <= 1e-5
    return y


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("length", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 333, 1000])
def test_one_token_of_one_sequence(qi, length, head_dim):
    attend(qi, Store(qi, length, [length], head_dim=head_dim), [0], [1], 8)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_of_every_size(qi, page):
    store = Store(qi, page, [5, 300, 64, 17], page=page)
    attend(qi, store, [2, 0, 3, 1], [1, 1, 1, 1], 2)
    attend(qi, store, [1, 3], [211, 17], 2)


@pytest.mark.parametrize("kv_heads,heads", [(1, 1), (1, 7), (3, 3), (2, 10), (4, 32), (1, 17), (5, 40)])
@pytest.mark.parametrize("most", [1, 3, 40])
def test_groups_of_heads(qi, kv_heads, heads, most):
    store = Store(qi, heads, [most, 77, 150, 200], kv_heads=kv_heads, head_dim=64 if heads == 10 else 128)
    attend(qi, store, [0, 1, 2, 3], [most, 1, most, min(most, 2)], heads)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("window", [0, 1, 15, 16, 100, 5000])
@pytest.mark.parametrize("counts", [[1, 1, 1], [5, 1, 8], [130, 300, 257]])
def test_masks(qi, causal, window, counts):
    attend(qi, Store(qi, window, [140, 650, 257]), [0, 1, 2], counts, 6, causal=causal, window=window)


@pytest.mark.parametrize("heads", [2, 16])
def test_rows_that_see_nothing(qi, heads):
    # sequences without a token, more queries than tokens, entries without a query
    store = Store(qi, 7, [0, 3, 20, 40, 400])
    attend(qi, store, [0, 1, 2, 3, 4], [1, 5, 0, 2, 1], heads)
    attend(qi, store, [0, 1, 2, 4], [30, 200, 300, 0], heads)
    attend(qi, store, [1, 0], [200, 4], heads, window=2)
    attend(qi, store, [0, 4], [1, 3], heads, causal=False)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("counts", [[4, 5, 2], [40, 300, 30]])
@pytest.mark.parametrize("window", [0, 2, 35])
def test_more_queries_than_tokens_without_a_causal_mask(qi, counts, window, head_dim):
    # rows before the first token see all of them, or with a window those that it reaches: zeros only where there are no tokens
    y = attend(qi, Store(qi, 49, [2, 34, 0], head_dim=head_dim), [0, 1, 2], counts, 4, causal=False, window=window)
    assert (y[: counts[0] + counts[1]] != 0).any(1).all() and (y[counts[0] + counts[1]:] == 0).all()


@pytest.mark.parametrize("window", [0x7fffffff, 0x7fffffff - 4, 1 << 30])
@pytest.mark.parametrize("counts", [[5, 6], [30, 290]])
@pytest.mark.parametrize("causal", [False, True])
def test_any_window(qi, window, counts, causal):
    # also for rows before the first token, whose positions are negative
    attend(qi, Store(qi, 29, [3, 280]), [0, 1], counts, 2, causal=causal, window=window)


def test_calls_of_different_shapes_share_a_workspace(qi):
    # counters of pieces lie where the partial results of another shape do not
    store = Store(qi, 31, [9000, 700, 3000, 40, 2500, 1200] + [900] * 58, page=64)
    dim, shapes = 128, [([0], [1], 2), (list(range(64)), [1] * 64, 16), ([2], [40], 2), (list(range(64)), [8] * 64, 2), ([0, 4], [33, 90], 6), (list(range(30)), [1] * 30, 2)]
    batches = [store.batch(slots, counts) for slots, counts, _ in shapes]
    workspace = torch.zeros(max(qi.kv_attention_workspace(store.cache, b, heads, 9000) for b, (_, _, heads) in zip(batches, shapes)), dtype=torch.uint8, device="cuda")
    for _ in range(2):
        for batch, (slots, counts, heads) in zip(batches, shapes):
            q = (torch.randn(sum(counts), heads, dim, device="cuda") * 1.5).half()
            y = torch.full_like(q, float("nan"))
            assert qi.kv_attention_ex(store.cache, store.pages, batch, store.layer, q, heads * dim, y, heads * dim, heads, dim ** -0.5, 9000, workspace=workspace) == 0
            settled(qi)
            exact, _ = attend_exact(store, q, slots, counts, heads, dim ** -0.5, True, 0)
            assert (y.double() - exact).norm() <= 2.0 ** -11 * exact.norm(), (counts, heads)


def test_a_workspace_for_the_largest_batch_serves_the_smaller_ones(qi):
    lengths, dim, heads = [5000, 900, 400, 70] * 10, 128, 8
    store = Store(qi, 39, lengths)
    largest = store.batch(list(range(40)), [900] * 40)
    workspace = torch.zeros(qi.kv_attention_workspace(store.cache, largest, heads, 5000), dtype=torch.uint8, device="cuda")
    for slots, counts in ((list(range(40)), [40] * 40), ([0], [900]), ([0, 2], [300, 300]), ([4], [5]), (list(range(40)), [1] * 40), ([8], [1]), ([0, 4, 8], [4, 2, 3])):
        q = (torch.randn(sum(counts), heads, dim, device="cuda") * 1.5).half()
        y, batch = torch.full_like(q, float("nan")), store.batch(slots, counts)
        for window in (0, 600):
            assert qi.kv_attention_ex(store.cache, store.pages, batch, 1, q, heads * dim, y, heads * dim, heads, dim ** -0.5, 5000, window=window, workspace=workspace) == 0
            settled(qi)
            exact, _ = attend_exact(store, q, slots, counts, heads, dim ** -0.5, True, window)
            assert (y.double() - exact).norm() <= 2.0 ** -11 * exact.norm(), (counts, window)


def test_the_example_serves_two_prompts_at_once(qi):
    import importlib.util

    spec = importlib.util.spec_from_file_location("cached_block_two", os.path.join(entry.ROOT, "examples", "cached_block.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    server = example.Server(qi, example.Model(qi))
    server.reserve([0, 1], [250, 262])
    assert torch.isfinite(server.forward([0, 1], [250, 262], torch.randn(512, example.WIDTH, device="cuda"))).all()
    assert all(word.item() == 0 for word in server.words)
    settled(qi)


def test_long_cache_is_split(qi):
    store = Store(qi, 3, [20011, 1, 9000], page=64)
    attend(qi, store, [0, 1, 2], [1, 1, 1], 8)
    attend(qi, store, [0, 2], [4, 2], 8)
    attend(qi, store, [0, 2], [150, 70], 8)
    attend(qi, store, [0], [1], 8, max_length=64 * store.table.shape[1])


@pytest.mark.parametrize("max_length", [0x7fffffff, 0x7fffffff - 127, 1 << 30, 1 << 27])
@pytest.mark.parametrize("slots,counts", [(list(range(40)), [20 + s % 13 for s in range(40)]), ([3, 7], [25, 20]), (list(range(40)), [1] * 40)], ids=["one piece", "pieces", "streaming"])
def test_any_bound_of_lengths(qi, max_length, slots, counts):
    # 80 units of rows leave one piece of the tokens for each, which is then as long as the bound
    attend(qi, Store(qi, 27, [50 + s for s in range(40)]), slots, counts, 2, max_length=max_length)


@pytest.mark.parametrize("lengths", [[rng % 301 for rng in range(0, 4000, 97)], [5, 0, 131, 9000, 1, 0, 700], [0, 0, 40, 0], [3000] * 5])
@pytest.mark.parametrize("entries", [2, 31, 129, 300])
def test_batches_of_many_entries(qi, lengths, entries):
    # more entries than threads, entries without queries or without tokens, short ones (a CTA to whole units) and long ones (units shared)
    rng = random.Random(entries + len(lengths))
    store = Store(qi, 9, lengths, kv_heads=1 if entries > 200 else 2)
    slots = [rng.randrange(len(lengths)) for _ in range(entries)]
    counts = [rng.choice((0, 1, 1, 1, 2)) for _ in slots]
    counts[0] = 1
    attend(qi, store, slots, counts, 4)


def test_many_queries(qi):
    store = Store(qi, 4, [1500, 1300, 129], page=64, kv_heads=2)
    attend(qi, store, [0, 1, 2], [1500, 700, 129], 4)
    attend(qi, store, [2, 1], [128, 1024], 2, causal=False)
    attend(qi, store, [1], [999], 14, window=300)


@pytest.mark.parametrize("kv_heads,heads", [(1, 7), (2, 2), (4, 12)])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 129), (False, 300), (True, 1)])
def test_many_queries_of_64_channels(qi, kv_heads, heads, causal, window):
    # several tiles of rows, which end within a tile of tokens, within a page and within a group of heads
    store = Store(qi, 51, [1100, 900, 257, 40], kv_heads=kv_heads, head_dim=64, page=32)
    attend(qi, store, [0, 1, 2, 3], [1100, 333, 257, 40], heads, causal=causal, window=window)
    attend(qi, store, [2, 1], [129, 513], heads, causal=causal, window=window)


@pytest.mark.parametrize("page", [16, 256])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_many_queries_over_a_long_cache_in_pieces(qi, head_dim, page):
    store = Store(qi, 53, [20011, 9000, 130], page=page, head_dim=head_dim, kv_heads=1)
    for causal, window in ((True, 0), (False, 0), (True, 5000), (False, 700)):
        attend(qi, store, [0, 1, 2], [150, 33, 130], 2, causal=causal, window=window)
        attend(qi, store, [1], [20], 1, causal=causal, window=window)


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("counts", [[1, 1], [3, 8], [90, 200]])
def test_queries_that_are_not_finite_spoil_their_own_rows_only(qi, counts, head_dim):
    store, heads, tokens = Store(qi, 55, [700, 260], head_dim=head_dim), 4, sum(counts)
    q = (torch.randn(tokens, heads, head_dim, device="cuda") * 1.5).half()
    exact, exact_lse = attend_exact(store, q, [0, 1], counts, heads, head_dim ** -0.5, True, 0)
    spoilt = torch.zeros(tokens, heads, dtype=torch.bool, device="cuda")
    for i, (token, head) in enumerate([(0, 1), (tokens - 1, 0), (tokens - 1, 3), (tokens // 2, 2)]):
        q[token, head, 5 * i] = (float("nan"), float("inf"), float("-inf"), float("nan"))[i]
        spoilt[token, head] = True
    y, lse, batch = torch.zeros_like(q), torch.zeros(tokens, heads, device="cuda"), store.batch([0, 1], counts)
    workspace = torch.zeros(qi.kv_attention_workspace(store.cache, batch, heads, 700), dtype=torch.uint8, device="cuda")
    assert qi.kv_attention_ex(store.cache, store.pages, batch, 1, q, heads * head_dim, y, heads * head_dim, heads, head_dim ** -0.5, 700, lse=lse, workspace=workspace) == 0
    settled(qi)
    assert y[spoilt].isnan().all()
    assert (y[~spoilt].double() - exact[~spoilt]).norm() <= 2.0 ** -11 * exact[~spoilt].norm() and (lse.double() - exact_lse)[~spoilt].abs().max() <= 1e-5


def test_strides_streams_and_loose_bounds(qi):
    store = Store(qi, 5, [500, 300])
    stream = torch.cuda.Stream()
    for counts in ([1, 1], [200, 33]):
        attend(qi, store, [1, 0], counts, 4, gap=24, stream=stream, max_length=900, most=max(counts) + 50)


@pytest.mark.parametrize("count", [1, 200])
def test_scales_that_differ_widely(qi, count):
    store = Store(qi, 6, [700])
    store.scales["v"][:, :, :, 0] *= 1000
    store.scales["v"][:, 3] = 0.0
    store.codes["v"][:, 3] = 128  # a page of zeros
    store.scales["k"][:, 5] = 0.0
    attend(qi, store, [0], [count], 4)
    for which in "kv":  # a dominant key far from the end
        store.codes[which][:, int(store.table[0, 2]), :, 5] = 255
    attend(qi, store, [0], [count], 4)


@pytest.mark.parametrize("counts", [[1, 1], [100, 300]])
def test_attention_in_a_graph_follows_lengths_on_the_device(qi, counts):
    store = Store(qi, 8, [700, 640])
    heads, dim = 4, 128
    batch = store.batch([0, 1], counts)
    q = torch.randn(sum(counts), heads, dim, device="cuda").half()
    y = torch.zeros_like(q)
    workspace = torch.zeros(qi.kv_attention_workspace(store.cache, batch, heads, 700), dtype=torch.uint8, device="cuda")
    call = lambda stream=None: qi.kv_attention_ex(store.cache, store.pages, batch, store.layer, q, heads * dim, y, heads * dim, heads, dim ** -0.5, 700, workspace=workspace, stream=stream)  # noqa: E731
    assert call() == 0
    settled(qi)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call(torch.cuda.current_stream().cuda_stream) == 0
    for lengths in ([700, 640], [650, 301], [400, 640]):
        store.lengths.copy_(ints(lengths))
        store.lengths_list = lengths
        graph.replay()
        settled(qi)
        exact, _ = attend_exact(store, q, [0, 1], counts, heads, dim ** -0.5, True, 0)
        assert (y.double() - exact).norm() <= 2.0 ** -11 * exact.norm()


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("counts", [[1, 1, 1, 1], [3, 8, 1, 2], [200, 30, 1, 150]])
@pytest.mark.parametrize("fault", [-1, -(1 << 31), 0x7fffffff, "pages"])
def test_attention_hides_tokens_without_a_page(qi, fault, counts, page, head_dim):
    # what no sound page holds enters no result: neither page 0, which may be another sequence's, nor what lay in shared memory before
    lengths, heads, group = [700, 330, 60, 150], 8, 4
    store = Store(qi, 33, lengths, page=page, head_dim=head_dim)
    for which in "kv":  # whatever is taken from elsewhere is large
        store.codes[which][:] = store.codes[which].where(torch.rand(store.codes[which].shape, device="cuda") < 0.5, 255 - store.codes[which].clamp(1, 254))
    held = [[which for which in range(-(-n // page))] for n in lengths]
    gone = [[0], [1, len(held[1]) - 1], held[2], [2]]  # the first, a middle and the last, all of them
    gone[0] += [j for j in held[0] if j % 3 == 2]
    k, v = ([store.values(which, s) for s in range(4)] for which in "kv")
    for s, missing in enumerate(gone):
        for j in missing:
            store.table[s, j] = len(store.references) if fault == "pages" else fault
    tokens = sum(counts)
    q = (torch.randn(tokens, heads, head_dim, device="cuda") * 1.5).half()
    batch, y, lse = store.batch([0, 1, 2, 3], counts), torch.full_like(q, float("nan")), torch.full((tokens, heads), float("nan"), device="cuda")
    workspace = torch.zeros(qi.kv_attention_workspace(store.cache, batch, heads, 700), dtype=torch.uint8, device="cuda")
    assert qi.kv_attention_ex(store.cache, store.pages, batch, 1, q, heads * head_dim, y, heads * head_dim, heads, head_dim ** -0.5, 700, lse=lse, workspace=workspace) == 0
    assert qi.kernel_status() >> 12 == 0x6C
    begin = 0
    for s, count in enumerate(counts):
        p, j = torch.arange(lengths[s] - count, lengths[s], device="cuda")[:, None], torch.arange(lengths[s], device="cuda")[None]
        hidden = (j > p) | torch.isin(j // page, torch.tensor(gone[s], device="cuda"))
        mine = q[begin:begin + count].double()
        scores = torch.einsum("ihd,jhd->hij", mine, k[s].repeat_interleave(group, 1)).mul(head_dim ** -0.5).masked_fill(hidden, -math.inf)
        exact_lse = scores.logsumexp(2)
        weights = torch.exp(scores - torch.where(exact_lse == -math.inf, 0.0, exact_lse)[..., None])
        exact = torch.einsum("hij,jhd->ihd", weights, v[s].repeat_interleave(group, 1))
        got, got_lse = y[begin:begin + count].double(), lse[begin:begin + count].T.double()
        begin += count
        seen = exact_lse > -math.inf
        assert torch.equal(got_lse > -math.inf, seen) and not got.isnan().any() and (got.transpose(0, 1)[~seen] == 0).all()
        assert (got - exact).abs().max() <= 2.0 ** -10 * v[s].abs().max() and (got - exact).norm() <= 2.0 ** -11 * exact.norm()
        if seen.any():
            assert (got_lse - exact_lse)[seen].abs().max() <= 1e-5


@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 200, 30]])
@pytest.mark.parametrize("fault", ["slot", "negative slot", "length", "negative length", "offset"])
def test_attention_and_read_leave_unsound_entries_alone(qi, fault, counts):
    lengths, heads, dim = [400, 250, 300], 4, 128
    store = Store(qi, 35, lengths, table_extra=8)
    batch, tokens, bad = store.batch([0, 1, 2], counts), sum(counts), 1
    q = (torch.randn(tokens, heads, dim, device="cuda") * 1.5).half()
    exact, exact_lse = attend_exact(store, q, [0, 1, 2], counts, heads, dim ** -0.5, True, 0)
    values = [torch.cat([store.values(which, s)[-n:] for s, n in zip((0, 1, 2), counts)]).float() for which in "kv"]
    if fault == "slot":
        batch.slots[1] = 3
    elif fault == "negative slot":
        batch.slots[1] = -1
    elif fault == "length":
        store.lengths[1] = 1 << 29  # more than a row of the table holds
    elif fault == "negative length":
        store.lengths[1] = -5
    else:
        batch.offsets[3], bad = tokens + 1, 2  # beyond the token rows
    y, lse = torch.full_like(q, float("nan")), torch.full((tokens, heads), float("nan"), device="cuda")
    out = torch.full((2, tokens, 2, dim), float("nan"), device="cuda")
    workspace = torch.zeros(qi.kv_attention_workspace(store.cache, batch, heads, 400), dtype=torch.uint8, device="cuda")
    assert qi.kv_attention_ex(store.cache, store.pages, batch, 1, q, heads * dim, y, heads * dim, heads, dim ** -0.5, 400, lse=lse, workspace=workspace) == 0
    assert qi.kernel_status() >> 12 == 0x6C
    assert qi.kv_read_ex(store.cache, store.pages, batch, 1, out[0], out[1], qi.DTYPE_F32, 2 * dim, 2 * dim) == 0
    assert qi.kernel_status() >> 12 == 0x6C
    for s in range(3):
        mine = slice(sum(counts[:s]), sum(counts[:s + 1]))
        if s == bad:
            assert y[mine].isnan().all() and lse[mine].isnan().all() and out[:, mine].isnan().all()
        else:
            assert (y[mine].double() - exact[mine]).norm() <= 2.0 ** -11 * exact[mine].norm() and (lse[mine].double() - exact_lse[mine]).abs().max() <= 1e-5
            assert all(torch.equal(out[i, mine], values[i][mine]) for i in range(2))


@pytest.mark.parametrize("fault", [-1, 0x7fffffff])
def test_read_leaves_rows_without_a_page_alone(qi, fault):
    store = Store(qi, 37, [100, 40], page=32)
    values = [torch.cat([store.values(which, s) for s in (0, 1)]).float() for which in "kv"]
    store.table[0, 1] = fault
    out = torch.full((2, 140, 2, 128), float("nan"), device="cuda")
    assert qi.kv_read_ex(store.cache, store.pages, store.batch([0, 1], [100, 40]), 1, out[0], out[1], qi.DTYPE_F32, 256, 256) == 0
    assert qi.kernel_status() >> 12 == 0x6C
    assert out[:, 32:64].isnan().all()
    for i in range(2):
        assert torch.equal(out[i, :32], values[i][:32]) and torch.equal(out[i, 64:], values[i][64:])


# ---- append and read back ------------------------------------------------------------------------------------------
#
# Codes and scales are equal to the definition's in 32 bits, bit for bit: products, divisions and roundings, each IEEE's.


def append_plain(store, kv, slots, counts):
    """The definition, block by block, on the CPU in float32."""
    begin = 0
    for s, count in zip(slots, counts):
        length = store.lengths_list[s]
        start = length - count
        for block in range(start // BLOCK, -(-length // BLOCK) if count else 0):
            first, end = max(start, block * BLOCK), min(length, (block + 1) * BLOCK)
            page = int(store.table[s, block * BLOCK // store.page])
            within = block * BLOCK % store.page
            for which, x in kv.items():
                new = x[begin + first - start:begin + end - start].float().cpu()
                codes, scales = store.codes[which][store.layer, page].cpu(), store.scales[which][store.layer, page].cpu()
                scale = new.abs().amax((0, 2)) * (1 / torch.tensor(127.0))
                early = first - block * BLOCK
                if early:
                    old = scales[:, within // BLOCK]
                    scale = torch.maximum(scale, old)
                    factor = torch.where(scale > 0, old / scale, torch.ones(()))
                    kept = codes[:, within:within + early].float() - 128
                    codes[:, within:within + early] = ((kept * factor[:, None, None]).round() + 128).to(torch.uint8)
                q = torch.where(scale[None, :, None] > 0, new / scale[None, :, None], torch.zeros(())).round().clamp(-127, 127) + 128
                codes[:, within + early:within + early + len(new)] = q.to(torch.uint8).transpose(0, 1)
                scales[:, within // BLOCK] = scale
                store.codes[which][store.layer, page], store.scales[which][store.layer, page] = codes.cuda(), scales.cuda()
        begin += count


def same_bytes(a, b):
    return all(torch.equal(a.codes[w], b.codes[w]) and torch.equal(a.scales[w].view(torch.int32), b.scales[w].view(torch.int32)) for w in "kv")


def make_kv(store, tokens, dtype, seed, gap=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    width = store.kv_heads * store.head_dim
    rows = torch.randn(tokens, 2 * width + gap, device="cuda", generator=g) * torch.exp2(torch.randn(tokens, 1, device="cuda", generator=g) * spread)
    rows = rows.to(dtype)
    return rows, {"k": rows[:, :width].view(tokens, -1, store.head_dim) if tokens else rows, "v": rows[:, width:2 * width].reshape(tokens, -1, store.head_dim) if tokens else rows}


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("head_dim,page,kv_heads", [(128, 32, 2), (64, 16, 3), (128, 256, 1), (64, 64, 5)])
def test_append_equals_the_definition_and_reads_back(qi, dtype, head_dim, page, kv_heads):
    lengths, counts, slots = [1, 16, 17, 100, 333, 64, 5], [1, 16, 1, 33, 300, 0, 3], [0, 1, 2, 3, 4, 5, 6]
    code = qi.DTYPE_F16 if dtype == torch.float16 else qi.DTYPE_F32
    a, b = (Store(qi, 11, lengths, kv_heads=kv_heads, head_dim=head_dim, page=page) for _ in range(2))
    rows, kv = make_kv(a, sum(counts), dtype, 12, gap=16)
    width, ld = kv_heads * head_dim, 2 * kv_heads * head_dim + 16
    append_plain(b, kv, slots, counts)
    for _ in range(2):  # writing the same tokens again changes nothing
        assert qi.kv_append_ex(a.cache, a.pages, a.batch(slots, counts), 1, rows, rows[:, width:], code, ld, ld) == 0
        settled(qi)
        assert same_bytes(a, b)
    out = torch.full((2, sum(counts), width + 8), float("nan"), dtype=dtype, device="cuda")
    assert qi.kv_read_ex(a.cache, a.pages, a.batch(slots, counts), 1, out[0], out[1], code, width + 8, width + 8) == 0
    settled(qi)
    assert out[:, :, width:].isnan().all()
    for i, which in enumerate("kv"):
        # one product in float32, rounded once more where the result is float16
        expected = torch.cat([a.values(which, s)[len(a.values(which, s)) - n:] for s, n in zip(slots, counts)]).float().to(dtype)
        assert torch.equal(out[i, :, :width].view(expected.shape), expected)


def test_append_token_by_token_into_fresh_pages(qi):
    # pages as an allocation leaves them: scales NaN, any codes. Scales only grow within a block, earlier tokens are rounded again.
    steps = 37
    a, b = (Store(qi, 13, [steps], page=16, fill=False) for _ in range(2))
    rows, kv = make_kv(a, steps, torch.float32, 14, spread=2.0)
    width = a.kv_heads * a.head_dim
    for t in range(1, steps + 1):
        for store in (a, b):
            store.lengths_list = [t]
            store.lengths.copy_(ints([t]))
        append_plain(b, {w: x[t - 1:t] for w, x in kv.items()}, [0], [1])
        assert qi.kv_append_ex(a.cache, a.pages, a.batch([0], [1]), 1, rows[t - 1:], rows[t - 1:, width:], qi.DTYPE_F32, 2 * width, 2 * width) == 0
    settled(qi)
    assert same_bytes(a, b)
    # the values are as near as codes of that scale can be: half a step from the last rounding, and half a step of each scale before it (at
    # most 15 times, each step no wider than the last one)
    held = a.values("k", 0)
    step = a.scales["k"][1].nan_to_num(0.0).max().double()  # the spare pages hold no token
    assert (held - kv["k"].double()).abs().max() <= 8 * step


def test_append_of_zeros_and_of_extremes(qi):
    store, plain = (Store(qi, 15, [16, 32], fill=False) for _ in range(2))
    rows, _ = make_kv(store, 48, torch.float32, 16)
    width = store.kv_heads * store.head_dim
    rows[:16] = 0.0
    rows[16:24] *= 1e30
    rows[24:32] *= 1e-30
    kv = {"k": rows[:, :width].view(48, -1, store.head_dim), "v": rows[:, width:].reshape(48, -1, store.head_dim)}
    append_plain(plain, kv, [0, 1], [16, 32])
    assert qi.kv_append_ex(store.cache, store.pages, store.batch([0, 1], [16, 32]), 1, rows, rows[:, width:], qi.DTYPE_F32, 2 * width, 2 * width) == 0
    settled(qi)
    assert same_bytes(store, plain)
    y = torch.zeros(1, 2, 128, dtype=torch.float16, device="cuda")
    assert qi.kv_attention_ex(store.cache, store.pages, store.batch([0], [1]), 1, torch.ones_like(y), 256, y, 256, 2, 1.0, 16) == 0
    settled(qi)
    assert (y == 0).all()


def test_what_rewriting_costs_a_prefix_in_the_same_block(qi):
    # Ten steps write other tokens behind 5 earlier ones of their block. Each growth of a scale rounds those once more, by half a step of the new scale;
    # a whole block ahead of them stays bit for bit; and what is written last is as near as a single rounding makes it.
    prefix, image, steps = 21, 30, 10
    store = Store(qi, 59, [prefix], page=16, spare=8, table_extra=2, fill=False)
    width = store.kv_heads * store.head_dim
    rows, kv = make_kv(store, prefix, torch.float32, 60, spread=0.0)
    assert qi.kv_append_ex(store.cache, store.pages, store.batch([0], [prefix]), 1, rows, rows[:, width:], qi.DTYPE_F32, 2 * width, 2 * width) == 0
    told, workspace = ints([9]), torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda")
    assert qi.kv_pages_reserve_ex(store.cache, store.pages, ints([0]), ints([image]), 1, told, workspace) == 0
    settled(qi)
    assert told.item() == 0
    first, growths, scale = store.values("k", 0)[:16].clone(), torch.ones(store.kv_heads, device="cuda"), None
    for step in range(steps):
        new, new_kv = make_kv(store, image, torch.float32, 61 + step, spread=0.5)
        assert qi.kv_append_ex(store.cache, store.pages, store.batch([0], [image]), 1, new, new[:, width:], qi.DTYPE_F32, 2 * width, 2 * width) == 0
        settled(qi)
        store.lengths_list = [prefix + image]
        now = store.scales["k"][1, int(store.table[0, 1]), :, 0].clone()
        growths += 1 if scale is None else (now > scale)  # the first step's counts, whether it grew or not
        assert scale is None or (now >= scale).all()
        scale = now
        held, bound = store.values("k", 0), (0.5 + 1e-4) * scale.double()
        assert torch.equal(held[:16], first)
        assert ((held[16:prefix] - kv["k"][16:].double()).abs() <= (growths * bound)[:, None]).all()
        assert ((held[prefix:32] - new_kv["k"][:32 - prefix].double()).abs() <= bound[:, None]).all()
    # appended again from the block's start, the prefix has its digits back
    both = torch.cat([rows[16:], new])
    assert qi.kv_append_ex(store.cache, store.pages, store.batch([0], [prefix - 16 + image]), 1, both, both[:, width:], qi.DTYPE_F32, 2 * width, 2 * width) == 0
    settled(qi)
    scale = store.scales["k"][1, int(store.table[0, 1]), :, 0].double()
    assert ((store.values("k", 0)[16:prefix] - kv["k"][16:].double()).abs() <= ((0.5 + 1e-4) * scale)[:, None]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_append_of_blocks_of_every_magnitude(qi, dtype):
    # a block each from the largest numbers down to those whose scale is no normal float32, or rounds to zero; then eight more tokens for each,
    # of which every other block's are larger, so that the earlier ones are rounded again by what may be a quotient of such scales
    sizes = [3e37, 1e30, 1.0, 2e-34, 1.2e-34, 1e-35, 1e-36, 1e-38, 1e-40, 1e-42, 2e-44, 0.0] if dtype == torch.float32 else [1e4, 1.0, 1e-3, 1e-4, 6e-6, 6e-8, 0.0]
    count = len(sizes)
    a, b = (Store(qi, 57, [8] * count, page=16, fill=False) for _ in range(2))
    width, code = a.kv_heads * a.head_dim, qi.DTYPE_F16 if dtype == torch.float16 else qi.DTYPE_F32
    g = torch.Generator(device="cuda").manual_seed(58)
    for step in range(2):
        rows = torch.randn(8 * count, 2 * width, device="cuda", generator=g).double().clamp(-4, 4)
        for i, size in enumerate(sizes):
            rows[8 * i:8 * i + 8] *= size * (2.5 if step and i % 2 else 1.0)
        rows = rows.to(dtype)
        for store in (a, b):
            store.lengths_list = [8 * (step + 1)] * count
            store.lengths.fill_(8 * (step + 1))
        append_plain(b, {"k": rows[:, :width].reshape(-1, a.kv_heads, a.head_dim), "v": rows[:, width:].reshape(-1, a.kv_heads, a.head_dim)}, list(range(count)), [8] * count)
        assert qi.kv_append_ex(a.cache, a.pages, a.batch(list(range(count)), [8] * count), 1, rows, rows[:, width:], code, 2 * width, 2 * width) == 0
        settled(qi)
        assert same_bytes(a, b), step
    if dtype == torch.float32:  # the blocks reach what is no normal number; float16 ones do not (2^-24 / 127)
        assert min(float(a.scales["k"][1, a.table[i, 0]].max()) for i, size in enumerate(sizes) if size) < 2.0 ** -126


@pytest.mark.parametrize("kv_heads", [1, 4, 9])
def test_append_and_read_without_a_bound_of_new_tokens(qi, kv_heads):
    lengths, counts = [333, 5, 40], [300, 1, 40]
    a, b = (Store(qi, 19, lengths, kv_heads=kv_heads, table_extra=2) for _ in range(2))
    rows, kv = make_kv(a, sum(counts), torch.float16, 20)
    width = a.kv_heads * a.head_dim
    append_plain(b, kv, [0, 1, 2], counts)
    batch = a.batch([0, 1, 2], counts, most=0x7fffffff)
    assert qi.kv_append_ex(a.cache, a.pages, batch, 1, rows, rows[:, width:], qi.DTYPE_F16, 2 * width, 2 * width) == 0
    out = torch.full((2, sum(counts), width), float("nan"), device="cuda")
    assert qi.kv_read_ex(a.cache, a.pages, batch, 1, out[0], out[1], qi.DTYPE_F32, width, width) == 0
    settled(qi)
    assert same_bytes(a, b)
    for i, which in enumerate("kv"):
        expected = torch.cat([a.values(which, s)[-n:] for s, n in zip((0, 1, 2), counts)]).float()
        assert torch.equal(out[i].view(expected.shape), expected)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_append_holds_what_is_not_finite_as_zero_and_says_so(qi, dtype, head_dim):
    lengths, counts = [1, 60, 333], [1, 41, 300]
    code = qi.DTYPE_F16 if dtype == torch.float16 else qi.DTYPE_F32
    a, b = (Store(qi, 43, lengths, head_dim=head_dim) for _ in range(2))
    rows, kv = make_kv(a, sum(counts), dtype, 44)
    width, g = a.kv_heads * head_dim, random.Random(45)
    places = [(0, 3), (1, width), (17, 2 * width - 1), (18, 0), (18, 1)] + [(g.randrange(20, 342), g.randrange(2 * width)) for _ in range(60)]
    places += [(200, c) for c in range(2 * width)]  # a token of nothing else
    clean = rows.clone()
    for i, (token, channel) in enumerate(places):
        rows[token, channel], clean[token, channel] = (float("nan"), float("inf"), float("-inf"))[i % 3], 0.0
    append_plain(b, {"k": clean[:, :width].reshape(-1, a.kv_heads, head_dim), "v": clean[:, width:].reshape(-1, a.kv_heads, head_dim)}, [0, 1, 2], counts)
    for _ in range(2):
        assert qi.kv_append_ex(a.cache, a.pages, a.batch([0, 1, 2], counts), 1, rows, rows[:, width:], code, 2 * width, 2 * width) == 0
        assert qi.kernel_status() & 0xfffff == 0x6C002
        assert same_bytes(a, b)
    assert qi.kv_append_ex(a.cache, a.pages, a.batch([0, 1, 2], counts), 1, clean, clean[:, width:], code, 2 * width, 2 * width) == 0
    settled(qi)


def test_append_leaves_shared_and_missing_pages_alone(qi):
    # page numbers are the device's own: what must not be written is left as it is, and the status word says so
    for fault in ("shared", "missing", "foreign", "count", "slot"):
        store, before = (Store(qi, 17, [20, 50]) for _ in range(2))
        batch = store.batch([0, 1], [4, 50])
        if fault == "shared":
            store.references[int(store.table[0, 0])] = 2
        elif fault == "missing":
            store.table[0, 0] = -1
        elif fault == "foreign":
            store.table[0, 0] = 1 << 30
        elif fault == "count":
            store.lengths[0] = 3
        else:
            batch.slots[0] = 2
        rows, kv = make_kv(store, 54, torch.float16, 18)
        append_plain(before, {w: x[4:] for w, x in kv.items()}, [1], [50])
        assert qi.kv_append_ex(store.cache, store.pages, batch, 1, rows, rows[:, 256:], qi.DTYPE_F16, 512, 512) == 0
        assert qi.kernel_status() >> 12 == 0x6C, fault
        assert same_bytes(store, before), fault
        assert qi.kernel_status() == 0


# ---- pages -----------------------------------------------------------------------------------------------------------


class Ledger:
    """What the page calls do, on the CPU: tables, lengths, references, and what each page holds."""

    def __init__(self, store):
        self.store, self.page = store, store.page
        self.table, self.lengths, self.references = store.table.tolist(), store.lengths.tolist(), store.references.tolist()
        self.content = list(range(len(self.references)))

    def free_pages(self):
        return [p for p, n in enumerate(self.references) if n == 0]

    def reserve(self, slots, counts):
        need = [-(-(self.lengths[s] + c) // self.page) - -(-self.lengths[s] // self.page) for s, c in zip(slots, counts)]
        free = self.free_pages()
        if sum(need) > len(free):
            return sum(need) - len(free)
        for s, c, n in zip(slots, counts, need):
            have = -(-self.lengths[s] // self.page)
            for j in range(have, have + n):
                self.table[s][j] = free.pop(0)
                self.references[self.table[s][j]] = 1
            self.lengths[s] += c
        return 0

    def fork(self, parents, children):
        old, lengths, free = [row[:] for row in self.table], self.lengths[:], self.free_pages()
        todo = [(p, c) for p, c in zip(parents, children) if p != c]
        need = sum(lengths[p] % self.page > 0 for p, _ in todo)
        if need > len(free):
            return need - len(free)
        content = self.content[:]
        for p, c in todo:
            for page in old[c]:
                if page >= 0:
                    self.references[page] -= 1
            whole, row = lengths[p] // self.page, [-1] * len(old[c])
            for j in range(whole):
                row[j] = old[p][j]
                self.references[row[j]] += 1
            if lengths[p] % self.page:
                row[whole] = free.pop(0)
                self.references[row[whole]] = 1
                self.content[row[whole]] = content[old[p][whole]]
            self.table[c], self.lengths[c] = row, lengths[p]
        return 0

    def free(self, slots):
        for s in slots:
            for page in self.table[s]:
                if page >= 0:
                    self.references[page] -= 1
            self.table[s], self.lengths[s] = [-1] * len(self.table[s]), 0

    def compact(self):
        used = sum(n > 0 for n in self.references)
        sources = [p for p, n in enumerate(self.references) if n > 0 and p >= used]
        targets = [p for p, n in enumerate(self.references) if n == 0 and p < used]
        for a, b in zip(sources, targets):
            self.references[b], self.references[a] = self.references[a], 0
            self.content[b] = self.content[a]
            self.table = [[b if page == a else page for page in row] for row in self.table]
        return used

    def check(self, start):
        store = self.store
        assert store.table.tolist() == self.table
        assert store.lengths.tolist() == self.lengths
        assert store.references.tolist() == self.references
        content = torch.tensor(self.content, device="cuda")
        for which in "kv":
            assert torch.equal(store.codes[which], start[which + "c"][:, content])
            assert torch.equal(store.scales[which].view(torch.int32), start[which + "s"][:, content].view(torch.int32))


def pool_copy(store):
    return {w + t: (store.codes if t == "c" else store.scales)[w].clone() for w in "kv" for t in "cs"}


@pytest.mark.parametrize("seed,page,layers,kv_heads,head_dim", [(1, 16, 1, 1, 64), (2, 32, 3, 2, 128), (3, 64, 2, 5, 64), (4, 256, 2, 8, 128)])
def test_pages_follow_the_ledger(qi, seed, page, layers, kv_heads, head_dim):
    rng = random.Random(seed)
    lengths = [rng.choice((0, 1, page - 1, page, page + 1, 3 * page, rng.randint(1, 5 * page))) for _ in range(23)]
    store = Store(qi, seed, lengths, page=page, layers=layers, layer=0, kv_heads=kv_heads, head_dim=head_dim, spare=29, table_extra=3)
    ledger, start = Ledger(store), pool_copy(store)
    workspace = torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda").fill_(0xA5)
    told = ints([77])
    for _ in range(12):
        what = rng.choice(("reserve", "fork", "fork", "free", "compact", "permute"))
        n = rng.randint(0, 9)
        slots = rng.sample(range(23), n)
        if what == "reserve":
            width = store.table.shape[1] * page
            slots = [s for s in slots if ledger.lengths[s] < width]
            counts = [min(rng.choice((0, 1, 2, page, 2 * page + 1)), width - ledger.lengths[s]) for s in slots]
            assert qi.kv_pages_reserve_ex(store.cache, store.pages, ints(slots + [0]), ints(counts + [0]), len(slots), told, workspace) == 0
            assert told.item() == ledger.reserve(slots, counts)
        elif what in ("fork", "permute"):
            parents = [rng.randrange(23) for _ in slots] if what == "fork" else rng.sample(slots, n)
            assert qi.kv_pages_fork_ex(store.cache, store.pages, ints(parents + [0]), ints(slots + [0]), n, told, workspace) == 0
            assert told.item() == ledger.fork(parents, slots)
        elif what == "free":
            assert qi.kv_pages_free_ex(store.cache, store.pages, ints(slots + [0]), n) == 0
            ledger.free(slots)
        else:
            assert qi.kv_pages_compact_ex(store.cache, store.pages, told, workspace) == 0
            assert told.item() == ledger.compact()
        settled(qi)
        ledger.check(start)


@pytest.mark.parametrize("counts", [[1, 1], [5, 1], [60, 33]])
def test_a_step_without_room_leaves_the_cache_alone(qi, counts):
    # the calls of a step are queued behind its reservation without waiting for it; where that falls short, "the last tokens" are earlier ones
    page, heads, dim = 16, 4, 128
    lengths = [32, 64, 80, 16]
    store, before = (Store(qi, 47, lengths, page=page, spare=1, table_extra=8) for _ in range(2))
    workspace = torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda")
    told, tokens = ints([5]), sum(counts)
    batch = qi.KvBatch(ints([0, 1]), ints([0, counts[0], tokens]), tokens, max(counts), told)
    rows, kv = make_kv(store, tokens, torch.float16, 48)
    q = (torch.randn(tokens, heads, dim, device="cuda") * 1.5).half()
    work = torch.zeros(max(qi.kv_attention_workspace(store.cache, batch, heads, 200), 16), dtype=torch.uint8, device="cuda")

    def step():
        y, lse, out = torch.full_like(q, float("nan")), torch.full((tokens, heads), float("nan"), device="cuda"), torch.full((2, tokens, 2, dim), float("nan"), device="cuda")
        assert qi.kv_pages_reserve_ex(store.cache, store.pages, ints([0, 1]), ints(counts), 2, told, workspace) == 0
        assert qi.kv_append_ex(store.cache, store.pages, batch, 1, rows, rows[:, 256:], qi.DTYPE_F16, 512, 512) == 0
        assert qi.kv_attention_ex(store.cache, store.pages, batch, 1, q, heads * dim, y, heads * dim, heads, dim ** -0.5, 200, lse=lse, workspace=work) == 0
        assert qi.kv_read_ex(store.cache, store.pages, batch, 1, out[0], out[1], qi.DTYPE_F32, 2 * dim, 2 * dim) == 0
        settled(qi)
        return y, lse, out

    y, lse, out = step()
    assert told.item() > 0 and store.lengths.tolist() == lengths
    assert same_bytes(store, before) and y.isnan().all() and lse.isnan().all() and out.isnan().all()
    told.fill_(-1)  # a list at fault likewise
    assert qi.kv_append_ex(store.cache, store.pages, batch, 1, rows, rows[:, 256:], qi.DTYPE_F16, 512, 512) == 0
    settled(qi)
    assert same_bytes(store, before)
    assert qi.kv_pages_free_ex(store.cache, store.pages, ints([2, 3]), 2) == 0
    y, lse, out = step()
    assert told.item() == 0
    store.lengths_list = before.lengths_list = [32 + counts[0], 64 + counts[1], 0, 0]
    before.table.copy_(store.table)
    append_plain(before, kv, [0, 1], counts)
    assert same_bytes(store, before)
    exact, _ = attend_exact(store, q, [0, 1], counts, heads, dim ** -0.5, True, 0)
    assert (y.double() - exact).norm() <= 2.0 ** -11 * exact.norm()
    assert torch.equal(out[0], torch.cat([store.values("k", s)[-n:] for s, n in zip((0, 1), counts)]).float())


def test_pages_that_do_not_suffice_change_nothing(qi):
    store = Store(qi, 5, [40, 64, 33], page=32, spare=1, table_extra=4)
    ledger, start = Ledger(store), pool_copy(store)
    workspace = torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda")
    told = ints([0])
    assert qi.kv_pages_reserve_ex(store.cache, store.pages, ints([0, 1]), ints([60, 1]), 2, told, workspace) == 0
    assert told.item() == 2
    ledger.check(start)
    assert qi.kv_pages_fork_ex(store.cache, store.pages, ints([0, 2]), ints([1, 0]), 2, told, workspace) == 0
    assert told.item() == 1
    ledger.check(start)
    settled(qi)
    # a list that is at fault: an unknown sequence, a negative count, more than a row of the table holds
    for slots, counts in (([3], [1]), ([-1], [1]), ([0], [-1]), ([0], [32 * store.table.shape[1]]), ([0], [0x7fffffff])):
        assert qi.kv_pages_reserve_ex(store.cache, store.pages, ints(slots), ints(counts), 1, told, workspace) == 0
        assert qi.kernel_status() >> 12 == 0x6C and told.item() == -1
    assert qi.kv_pages_fork_ex(store.cache, store.pages, ints([0]), ints([9]), 1, told, workspace) == 0
    assert qi.kernel_status() >> 12 == 0x6C and told.item() == -1
    assert qi.kv_pages_free_ex(store.cache, store.pages, ints([9]), 1) == 0
    assert qi.kernel_status() >> 12 == 0x6C
    ledger.check(start)


@pytest.mark.parametrize("fault", [-1, 0x7fffffff])
def test_a_fork_of_a_sequence_whose_last_page_is_missing(qi, fault):
    # the child has no page there either, not a free one with what it last held; the other children of the call are as always
    store = Store(qi, 63, [75, 40, 10, 5], page=32, spare=6, table_extra=2)
    store.table[0, 2] = fault
    rows, references, start = store.table.tolist(), store.references.tolist(), pool_copy(store)
    told, workspace = ints([9]), torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda").fill_(0xA5)
    assert qi.kv_pages_fork_ex(store.cache, store.pages, ints([0, 1]), ints([2, 3]), 2, told, workspace) == 0
    assert qi.kernel_status() >> 12 == 0x6C
    assert told.item() == 0 and store.lengths.tolist() == [75, 40, 75, 40]
    table, now = store.table.tolist(), store.references.tolist()
    free = [p for p, n in enumerate(references) if n == 0]
    assert table[:2] == rows[:2]
    assert table[2] == rows[0][:2] + [-1] * (len(rows[0]) - 2)
    assert table[3][0] == rows[1][0] and table[3][1] in free[:2] and table[3][2:] == [-1] * (len(rows[0]) - 2)
    for p in rows[0][:2] + [rows[1][0]]:
        references[p] += 1
    for p in (rows[2][0], rows[3][0]):
        references[p] -= 1
    references[table[3][1]] = 1
    assert now == references
    for which in "kv":
        expected = start[which + "c"].clone()
        expected[:, table[3][1]] = expected[:, rows[1][1]]
        assert torch.equal(store.codes[which], expected)


def test_reserving_for_a_sequence_twice_stays_within_its_row(qi):
    # against the rules, and what it gives is not defined, but other rows, what lies behind the table and other pages are left alone
    page, sequences, width = 16, 40, 3
    store = Store(qi, 41, [32] * sequences, page=page, spare=50, table_extra=1)
    whole = torch.full((sequences * width + 64,), 1234567, dtype=torch.int32, device="cuda")
    whole[: sequences * width] = store.table.flatten()
    table = whole[: sequences * width].view(sequences, width)
    pages = qi.KvPages(table, store.lengths, store.references)
    workspace = torch.empty(qi.kv_pages_workspace(store.cache, pages), dtype=torch.uint8, device="cuda").fill_(0xA5)
    told, last = ints([0]), sequences - 1
    slots = [last] + list(range(31)) + [last] + [31, 32]  # the first and the 33rd of the list are one warp's, one after the other
    assert qi.kv_pages_reserve_ex(store.cache, pages, ints(slots), ints([16] * len(slots)), len(slots), told, workspace) == 0
    settled(qi)
    assert told.item() == 0
    assert (whole[sequences * width:] == 1234567).all()
    assert ((table >= -1) & (table < len(store.references))).all() and (store.lengths <= width * page).all()
    for s in range(33):
        assert store.lengths[s] == 48 and table[s, 2] >= 0
    for s in range(33, last):
        assert store.lengths[s] == 32 and table[s, 2] == -1
    held = table[table >= 0]
    assert len(held.unique()) == len(held)


def test_pages_of_a_large_pool(qi):
    # more pages than one round of the planning CTA looks at, and a compaction that moves most of them
    store = Store(qi, 6, [16 * 9] * 700, page=16, layers=1, layer=0, kv_heads=1, head_dim=64, spare=6000, table_extra=2)
    ledger, start = Ledger(store), pool_copy(store)
    workspace = torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda")
    told = ints([0])
    gone = list(range(0, 700, 3))
    assert qi.kv_pages_free_ex(store.cache, store.pages, ints(gone), len(gone)) == 0
    ledger.free(gone)
    assert qi.kv_pages_compact_ex(store.cache, store.pages, told, workspace) == 0
    assert told.item() == ledger.compact()
    more = list(range(700))
    assert qi.kv_pages_reserve_ex(store.cache, store.pages, ints(more), ints([17] * 700), 700, told, workspace) == 0
    assert told.item() == ledger.reserve(more, [17] * 700) == 0
    settled(qi)
    ledger.check(start)


def test_copying_pages(qi):
    store = Store(qi, 7, [300], page=32, layers=3)
    start = pool_copy(store)
    assert qi.kv_pages_copy_ex(store.cache, ints([0, 3, 5]), ints([1, 4, 2]), 3) == 0
    settled(qi)
    for which in "kv":
        for kind, now in (("c", store.codes[which]), ("s", store.scales[which])):
            expected = start[which + kind].clone()
            expected[:, [1, 4, 2]] = start[which + kind][:, [0, 3, 5]]
            assert torch.equal(now.view(torch.uint8), expected.view(torch.uint8))
    assert qi.kv_pages_copy_ex(store.cache, ints([0]), ints([99]), 1) == 0
    assert qi.kernel_status() >> 12 == 0x6C


# ---- norms -----------------------------------------------------------------------------------------------------------
#
# Tolerance. Everything is float32 but the stores: sums of w squares in a tree of at most 64 serial additions, 2^-18 of a positive sum, so a norm's
# factor is within 2^-18; a handful of products and sums after it, 2^-22 each. With two norms in a row: 2^-16 of the largest term in magnitude.
# float16 results add half a unit, 2^-11.


def norm_exact(x, kind, epsilon, qi):
    if kind == qi.NORM_LAYER:
        x = x - x.mean(-1, keepdim=True)
    return x / (x.square().mean(-1, keepdim=True) + epsilon).sqrt()


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,width", [(1, 8), (3, 64), (5, 1000), (2, 1024), (7, 2048), (300, 3080), (2, 4096), (9, 5120), (3, 8200), (2, 16384), (3000, 512), (1700, 768), (4, 1016), (950, 1280), (5, 1288), (700, 1536), (500, 2504), (3, 2560), (350, 3072), (200, 6144)])
def test_norms(qi, kind, rows, width):
    kind = qi.NORM_LAYER if kind == "layer" else qi.NORM_RMS
    g = torch.Generator(device="cuda").manual_seed(rows + width)
    code = {torch.float16: qi.DTYPE_F16, torch.float32: qi.DTYPE_F32}
    for case in range(6):
        residual_type, branch_type, vector_type, y_type = (torch.float16 if case >> i & 1 else torch.float32 for i in range(4))
        if case == 5:
            residual_type, branch_type, vector_type, y_type = torch.float32, torch.float16, torch.float16, torch.float32
        normal = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
        residual, branch = (normal(rows, width) * 4 + 2).to(residual_type), (normal(rows, width) * 7 - 3).to(branch_type)
        groups = 1 if case % 2 else 3
        each = -(-rows // groups)
        vectors = (normal(groups, 3 * width + 8) * 0.3).to(vector_type)
        gate, scale, shift = (vectors[:, i * width:] if case != 2 else None for i in range(3))
        branch_norm, weight = case in (0, 3, 5), normal(width) if case in (0, 1) else None
        branch_weight = normal(width) if case in (0, 4) else None
        out, y = torch.full_like(residual, float("nan")), torch.full((rows, width), float("nan"), dtype=y_type, device="cuda")
        call = qi.GatedNorm(rows, width, kind=kind, epsilon=1e-5, residual=residual, residual_dtype=code[residual_type], branch=branch, branch_dtype=code[branch_type],
                            branch_norm=branch_norm, branch_weight=branch_weight, residual_scale=0.7, gate=gate, scale=scale, shift=shift, vector_dtype=code[vector_type],
                            ld_vector=3 * width + 8, rows_per_vector=each, weight=weight, residual_out=out, y=y, y_dtype=code[y_type])
        assert qi.gated_norm_ex(call) == 0
        settled(qi)
        owner = torch.arange(rows, device="cuda") // each
        b = branch.double()
        if branch_norm:
            b = norm_exact(b, kind, 1e-5, qi)
        if branch_weight is not None:
            b = b * branch_weight.double()
        if gate is not None:
            b = b * gate[owner, :width].double()
        r = residual.double() + float(torch.tensor(0.7)) * b
        n = norm_exact(r, kind, 1e-5, qi)
        if weight is not None:
            n = n * weight.double()
        terms = n.abs()
        if scale is not None:
            n = n * (1 + scale[owner, :width].double())
            terms = n.abs() + shift[owner, :width].double().abs()
            n = n + shift[owner, :width].double()
        for got, exact, size, dtype in ((out, r, residual.double().abs() + b.abs(), residual_type), (y, n, terms, y_type)):
            bound = 2.0 ** -16 * size.amax(-1, keepdim=True) + (2.0 ** -11 * exact.abs() if dtype == torch.float16 else 0.0)
            assert ((got.double() - exact).abs() <= bound).all(), (case, dtype)


def test_norm_alone_in_place_and_on_another_stream(qi):
    x, branch = torch.randn(50, 4096, device="cuda"), torch.randn(50, 4096, device="cuda")
    expected, y = x + branch, torch.empty(50, 4096, dtype=torch.float16, device="cuda")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    assert qi.gated_norm_ex(qi.GatedNorm(50, 4096, residual=x, branch=branch, residual_out=x, y=y, y_dtype=qi.DTYPE_F16), stream.cuda_stream) == 0
    settled(qi)
    assert torch.equal(x, expected)
    alone = torch.empty_like(y)
    assert qi.gated_norm_ex(qi.GatedNorm(50, 4096, residual=x, y=alone, y_dtype=qi.DTYPE_F16)) == 0
    assert qi.gated_norm_ex(qi.GatedNorm(50, 4096, residual=x, branch=branch, residual_out=x)) == 0
    settled(qi)
    assert torch.equal(alone, y) and torch.equal(x, expected + branch)


def test_norm_of_rows_without_spread(qi):
    # a constant row has no deviation: epsilon keeps it finite; a large mean costs no digits of what is left
    x = torch.full((3, 2048), 5.0, device="cuda")
    x[1] = 0.0
    x[2] = 1e4 + torch.randn(2048, device="cuda")
    y = torch.empty_like(x)
    assert qi.gated_norm_ex(qi.GatedNorm(3, 2048, kind=qi.NORM_LAYER, residual=x, y=y)) == 0
    settled(qi)
    assert (y[:2] == 0).all()
    exact = norm_exact(x[2:].double(), qi.NORM_LAYER, 1e-6, qi)
    assert (y[2:].double() - exact).abs().max() <= 2.0 ** -10  # a mean of 1e4 in 32 bits is known to 2^-11 of a deviation


@pytest.mark.parametrize("kind", ["layer", "rms"])
@pytest.mark.parametrize("rows,width", [(700, 512), (900, 4096), (5, 16384)])
def test_rows_that_are_not_finite_spoil_themselves_only(qi, kind, rows, width):
    kind = qi.NORM_LAYER if kind == "layer" else qi.NORM_RMS
    x, branch, weight = torch.randn(rows, width, device="cuda"), torch.randn(rows, width, device="cuda").half(), torch.randn(width, device="cuda")

    def call():
        y, out = torch.empty(rows, width, device="cuda"), torch.empty(rows, width, device="cuda")
        assert qi.gated_norm_ex(qi.GatedNorm(rows, width, kind=kind, residual=x, branch=branch, branch_dtype=qi.DTYPE_F16, branch_norm=True, weight=weight, residual_out=out, y=y)) == 0
        settled(qi)
        return y, out

    clean = call()
    x[1, 7], branch[rows - 2, 100], x[rows // 2, width - 1] = float("nan"), float("inf"), float("-inf")
    spoilt = torch.zeros(rows, dtype=torch.bool, device="cuda")
    spoilt[[1, rows - 2, rows // 2]] = True
    for now, before in zip(call(), clean):
        assert torch.equal(now[~spoilt], before[~spoilt])
        assert now[spoilt].isfinite().all(1).logical_not().all()


# ---- together ----------------------------------------------------------------------------------------------------------


def test_the_example_runs_and_both_ways_agree(qi):
    # Token by token, blocks of 16 tokens are rounded again as their scales grow: keys and values differ by a code or so, half a percent of a
    # deviation, from those appended at once; an attention's result by about as much, and three blocks add that up to a few percent at
    # most. Wrong pages, positions or masks give outputs that have nothing in common (1.4 apart).
    import importlib.util

    spec = importlib.util.spec_from_file_location("cached_block", os.path.join(entry.ROOT, "examples", "cached_block.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    difference, stepwise = example.main()
    assert difference <= 0.1
    assert torch.isfinite(stepwise).all()


def test_block_scales_of_shared_prompts_are_the_parents(qi):
    # a fork reads the prompt that its parent appended: same attention, bit for bit, from shared pages and from the copied last one
    store = Store(qi, 21, [75, 0, 0], page=32, spare=8, table_extra=2)
    workspace = torch.empty(qi.kv_pages_workspace(store.cache, store.pages), dtype=torch.uint8, device="cuda")
    told = ints([9])
    assert qi.kv_pages_fork_ex(store.cache, store.pages, ints([0, 0]), ints([1, 2]), 2, told, workspace) == 0
    assert told.item() == 0
    store.lengths_list = [75, 75, 75]
    q = (torch.randn(1, 4, 128, device="cuda") * 1.5).half().expand(3, -1, -1).contiguous()
    y = attend(qi, store, [0, 1, 2], [1, 1, 1], 4, q=q)
    assert torch.equal(y[0], y[1]) and torch.equal(y[0], y[2])
