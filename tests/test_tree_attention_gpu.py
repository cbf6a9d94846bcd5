"""Attention over a paged cache against float64, at the sizes, masks and layouts where a kernel can go wrong."""
import math

import pytest
import torch

from hf_rocm_kernels import append_kv, rotary_frequencies, tree_attention
from oracle import attention as oracle

pytestmark = pytest.mark.gpu

FP8 = torch.float8_e4m3fn
LONG = 1 << 20  # places in a table's row with which a call counts as much work, whatever the lengths are: many rows take the kernel with LDS


class Step:
    """A step's queries and the cache they read, on the CPU: pages in a random order, memory that nobody may read filled with NaN."""

    def __init__(self, lengths, counts, heads, kv_heads, head_dim, page, dtype=torch.bfloat16, cache=None, layout="tokens", tree=None, seed=0, extra=0,
                 uniform=False, loud=1.0, places=0):
        g = self.g = torch.Generator().manual_seed(seed)
        cache = cache or dtype
        self.dtype, self.cache, self.lengths, self.counts = dtype, cache, lengths, counts
        seqs, total = len(lengths), sum(counts)
        need = [-(-n // page) for n in lengths]
        columns = max(max(need) + 1, places // page, 2)
        order = torch.randperm(sum(need) + 3, generator=g).tolist()
        pages = len(order)
        self.table = torch.full((seqs, columns), -1, dtype=torch.int32)
        for b, n in enumerate(need):
            for i in range(n):
                self.table[b, i] = order.pop()
        shape = (pages, kv_heads, page, head_dim) if layout == "heads" else (pages, page, kv_heads, head_dim)
        caches = [torch.full(shape, math.nan).to(cache) for _ in range(2)]
        if layout == "heads":
            caches = [c.transpose(1, 2) for c in caches]
        for c in caches:
            bytes_ = c.view(torch.uint8) if cache == FP8 else c
            for b, n in enumerate(lengths):
                for i in range(need[b]):
                    rows = min(page, n - i * page)
                    x = torch.randn(rows, kv_heads, head_dim, generator=g) * (60.0 if cache == FP8 else 1.0)
                    x = x.clamp(-448, 448).to(cache)
                    bytes_[int(self.table[b, i]), :rows] = x.view(torch.uint8) if cache == FP8 else x
        self.key, self.value = caches
        self.layout = layout
        self.query = (torch.randn(total + extra, heads, head_dim, generator=g) * loud).to(dtype)
        self.starts = None if uniform else torch.tensor([sum(counts[:b]) for b in range(seqs + 1)], dtype=torch.int32)
        self.mask = None
        if tree is not None:
            width = max(counts) if tree == "full" else tree if isinstance(tree, int) else max(counts)
            sees = torch.rand(total + extra, max(width, 1), generator=g) < 0.4
            self.mask = sees[:, :width] if width else sees[:, :0]
        self.key_scale = self.value_scale = None
        if cache == FP8:
            self.key_scale = torch.rand(kv_heads, generator=g) * 0.02 + 0.01
            self.value_scale = torch.tensor([0.0173])
        self.scale = 1.0 / math.sqrt(head_dim)

    def args(self):
        def up(t):
            return None if t is None else t.cuda()
        # (.cuda() keeps a transposed view's strides)
        return dict(query=up(self.query), key_cache=up(self.key), value_cache=up(self.value), page_table=up(self.table),
                    lengths=torch.tensor(self.lengths, dtype=torch.int32, device="cuda"), starts=up(self.starts), mask=up(self.mask),
                    key_scale=up(self.key_scale), value_scale=up(self.value_scale))

    def check(self, got, out_scale=None, lengths=None):
        found = oracle.attention(self.query, self.key, self.value, self.table, torch.tensor(lengths or self.lengths), self.starts, self.mask, self.scale,
                                 self.key_scale, self.value_scale)
        want = found[0]
        got = got.cpu().double() * (1.0 if out_scale is None else out_scale)
        rows = sum(self.counts)
        tol = oracle.attention_tolerance(found, self.dtype, max(max(self.lengths), 1), None if out_scale is None else FP8, out_scale or 1.0)[:rows]
        want, got = want[:rows], got[:rows]
        if out_scale is not None:
            want = want.clamp(-448 * out_scale, 448 * out_scale)
        fine = torch.isfinite(want)
        assert torch.equal(fine, torch.isfinite(got)), "infinities or NaN in other places"
        assert torch.equal(torch.isnan(want), torch.isnan(got)) and torch.equal(want[~fine & ~torch.isnan(want)], got[~fine & ~torch.isnan(got)])
        off = (got - want).abs()[fine]
        worst = float((off / tol[fine]).max()) if off.numel() else 0.0
        assert worst <= 1.0, worst


TYPES = [(torch.bfloat16, None), (torch.float16, None), (torch.bfloat16, FP8), (torch.float16, FP8)]


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("head_dim", [16, 64, 80, 96, 128, 144, 256])
def test_one_token_of_each_length(dtype, cache, head_dim):
    """Lengths around every boundary: a lane's eight tokens, a wave's 32, a workgroup's 128, a page's end, a split."""
    lengths = [1, 7, 8, 9, 31, 32, 33, 64, 127, 128, 129, 200, 257, 0, 16, 500]
    step = Step(lengths, [1] * len(lengths), 8, 2, head_dim, 24, dtype, cache, uniform=True, seed=head_dim)
    step.check(tree_attention(**step.args()))


@pytest.mark.parametrize("head_dim", [40, 72, 104])
def test_heads_that_end_inside_a_window(head_dim):
    step = Step([100, 33], [1, 1], 6, 3, head_dim, 16, torch.float16, uniform=True, layout="heads")
    step.check(tree_attention(**step.args()))


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (4, 4), (32, 8), (5, 1), (35, 5), (14, 2), (16, 1), (48, 2)])
@pytest.mark.parametrize("page,layout", [(8, "tokens"), (16, "heads"), (40, "tokens"), (1000, "heads")])
def test_head_groups_and_pages(heads, kv_heads, page, layout):
    step = Step([130, 77, 300], [1, 1, 1], heads, kv_heads, 64, page, torch.bfloat16, layout=layout, seed=heads)
    step.check(tree_attention(**step.args()))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("counts", [[3, 1, 5], [9, 16, 1, 0, 7], [27, 40], [70, 1, 0, 33]])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("places", [0, LONG])
def test_chains_and_trees(dtype, cache, head_dim, counts, tree, places):
    """Blocks of 16, 32, 128 and 256 rows, the last of a sequence ragged; sequences with no token, masks with empty rows, rows of nobody behind the last."""
    lengths = [n + 37 * (i + 1) for i, n in enumerate(counts)]
    lengths[0] = counts[0]  # nothing in front of the step: rows that see nothing
    step = Step(lengths, counts, 8, 2, head_dim, 16, dtype, cache, tree="full" if tree else None, seed=sum(counts), extra=2, places=places)
    if tree:
        step.mask[1] = False
    out = torch.full(step.query.shape, 7.0, dtype=dtype, device="cuda")
    got = tree_attention(**step.args(), output=out)
    assert got.data_ptr() == out.data_ptr()
    step.check(got)
    assert (got[sum(counts):] == 7.0).all()


@pytest.mark.parametrize("seqs,most", [(70, 1), (130, 3), (3, 1)])
def test_many_sequences(seqs, most):
    """More sequences than a wave has lanes; some empty, one much longer than the others."""
    g = torch.Generator().manual_seed(seqs)
    counts = torch.randint(0, most + 1, (seqs,), generator=g).tolist()
    lengths = [0 if n == 0 and i % 2 else n + int(torch.randint(0, 40, (1,), generator=g)) for i, n in enumerate(counts)]
    counts[seqs // 2], lengths[seqs // 2] = most, 1500
    step = Step(lengths, counts, 4, 2, 64, 16, torch.float16, seed=seqs)
    step.check(tree_attention(**step.args()))


@pytest.mark.parametrize("dtype,cache", TYPES)
@pytest.mark.parametrize("counts,length", [([1], 5000), ([20], 3000), ([6, 1], 2500)])
@pytest.mark.parametrize("places", [0, LONG])
def test_long_caches_split_between_workgroups(dtype, cache, counts, length, places):
    lengths = [length - 700 * i for i in range(len(counts))]
    step = Step(lengths, counts, 4, 1, 128, 32, dtype, cache, seed=length, loud=3.0, places=places)
    first = tree_attention(**step.args())
    step.check(first)
    again = tree_attention(**step.args())
    assert torch.equal(first, again)  # equal calls, equal bits


@pytest.mark.parametrize("dtype,cache", [(torch.bfloat16, None), (torch.float16, FP8)])
@pytest.mark.parametrize("counts,places", [([2, 5, 1], 0), ([2, 50, 1], LONG)])
def test_output_in_fp8(dtype, cache, counts, places):
    step = Step([300, 20 if places == 0 else 60, 0], counts, 8, 2, 128, 16, dtype, cache, seed=4, places=places)
    for s in (0.004, 0.0002):  # the second saturates
        got = tree_attention(**step.args(), out_scale=torch.tensor([s], device="cuda"))
        assert got.dtype == FP8
        step.check(got.float(), out_scale=float(torch.tensor(s)))


@pytest.mark.parametrize("heads,places", [(4, 0), (32, LONG)])
def test_a_step_longer_than_its_cache_and_pages_that_are_missing(heads, places):
    step = Step([3, 90, 60, 50], [6, 2, 2, 4], heads, 2, 64, 16, seed=2, places=places)
    step.table[1, 2] = -1          # a hole
    step.table[2, :] = 10 ** 6     # no page of it exists: zeros
    step.table[3, 0] = -2147483648
    step.lengths[3] = 10 ** 9      # longer than its row of the table
    step.lengths[1] = 89
    args = step.args()
    got = tree_attention(**args)
    step.check(got)
    assert (got[8:10] == 0).all()


@pytest.mark.parametrize("width", [0, 2])
@pytest.mark.parametrize("counts,places", [([5, 6], 0), ([30, 26], LONG)])
def test_masks_with_fewer_columns_than_the_step(width, counts, places):
    step = Step([40, counts[1]], counts, 4, 2, 64, 16, tree=width, seed=6, places=places)
    step.check(tree_attention(**step.args()))
    step.mask = (step.mask * 255).to(torch.uint8)  # bytes, any but zero
    step.check(tree_attention(**step.args()))


@pytest.mark.parametrize("dtype,cache,what", [(d, None, w) for d in (torch.bfloat16, torch.float16) for w in (math.nan, math.inf, -math.inf)] +
                         [(torch.bfloat16, FP8, math.nan)])  # (e4m3fn has no infinities)
@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("places", [0, LONG])
def test_infinities_and_nan_of_drafted_tokens_reach_only_those_who_see_them(dtype, cache, what, head_dim, places):
    for counts in ([5, 1], [20, 3], [40]):
        step = Step([n + 30 for n in counts], counts, 4, 2, head_dim, 8, dtype, cache, tree="full", seed=9, places=places)
        token = step.lengths[0] - counts[0] + 2  # the third drafted token
        page, place = int(step.table[0, token // 8]), token % 8
        if cache == FP8:
            step.value.view(torch.uint8)[page, place, 1, 3] = 0x7f
        else:
            step.value[page, place, 1, 3] = what
        for i in range(counts[0]):
            step.mask[i, 2] = i % 2 == 0
        step.check(tree_attention(**step.args()))
        # a key that nobody sees
        step.mask[:counts[0], 2] = False
        step.key.view(torch.uint8)[page, place] = 0x7f
        if cache is None:
            step.key[page, place] = what
        step.check(tree_attention(**step.args()))


def test_a_weight_that_underflows_and_scores_far_apart():
    step = Step([200], [3], 4, 2, 64, 16, torch.float16, seed=3, loud=60.0)
    step.check(tree_attention(**step.args()))


def test_strides():
    """A projection's slice as the query, keys and values of a page in one tensor, a table and a mask cut from wider ones."""
    step = Step([100, 45], [4, 3], 8, 2, 64, 16, tree="full", seed=12)
    args = step.args()
    want = tree_attention(**args)
    step.check(want)
    rows = torch.zeros(7, 13, 64, dtype=torch.bfloat16, device="cuda")
    rows[:, 2:10] = args["query"]
    both = torch.stack((args["key_cache"], args["value_cache"]), dim=1)
    table = torch.full((2, 50), -7, dtype=torch.int32, device="cuda")
    table[:, 3:3 + step.table.shape[1]] = args["page_table"]
    mask = torch.ones(7, 30, dtype=torch.bool, device="cuda")
    mask[:, 5:5 + step.mask.shape[1]] = args["mask"]
    wide = torch.zeros(7, 20, 64, dtype=torch.bfloat16, device="cuda")
    got = tree_attention(rows[:, 2:10], both[:, 0], both[:, 1], table[:, 3:3 + step.table.shape[1]], args["lengths"], args["starts"],
                         mask[:, 5:5 + step.mask.shape[1]], output=wide[:, 4:12])
    assert torch.equal(got, want) and not wide[:, :4].any() and not wide[:, 12:].any()
    by_heads = args["query"].transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(tree_attention(**{**args, "query": by_heads}), want)


def test_offsets_past_32_bits():
    memory = torch.zeros(2, 3, 1 << 30, dtype=torch.bfloat16, device="cuda")
    far = [memory[i].view(-1).as_strided((3, 16, 2, 64), (1 << 30, 128, 64, 1)) for i in range(2)]
    step = Step([40], [2], 4, 2, 64, 16, seed=1)
    args = step.args()
    used = step.table[0, :3].tolist()
    for c, name in zip(far, ("key_cache", "value_cache")):
        for i, p in enumerate(used):
            c[i] = args[name][p]
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
    got = tree_attention(**{**args, "key_cache": far[0], "value_cache": far[1], "page_table": table})
    assert torch.equal(got, tree_attention(**args))


@pytest.mark.parametrize("pages_far", [True, False])
@pytest.mark.parametrize("counts", [[2], [70]])
def test_wide_strides(pages_far, counts):
    """Strides of pages that 32 bits just hold in bytes, strides of places that they do not: the kernels of few and of many rows."""
    step = Step([100], counts, 4, 2, 64, 8 if not pages_far else 16, seed=2, places=LONG if counts == [70] else 0)
    args = step.args()
    pages = step.key.size(0)
    far = {}
    for name in ("key_cache", "value_cache"):
        if pages_far:
            strides = (1 << 30, 128, 64, 1)
            memory = torch.zeros(((pages - 1) << 30) + 16 * 128, dtype=torch.bfloat16, device="cuda")
        else:
            strides = (128, 1 << 27, 64, 1)
            memory = torch.zeros(8 << 27, dtype=torch.bfloat16, device="cuda")
        far[name] = memory.as_strided(step.key.shape, strides)
        far[name].copy_(args[name])
    assert torch.equal(far["key_cache"].nan_to_num(7.0), args["key_cache"].nan_to_num(7.0))
    got = tree_attention(**{**args, **far})
    if pages_far or sum(counts) == 2:
        assert torch.equal(got, tree_attention(**args))  # the same kernel: the same bits
    step.check(got)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("head_dim", [64, 128])
def test_many_rows_in_graphs_on_two_streams(head_dim, tree):
    """The kernel of many rows: two captured calls replayed at once, with other lengths, pages and masks than at the capture."""
    step = Step([2000, 700], [50, 90], 8, 2, head_dim, 16, tree="full" if tree else None, seed=6, places=LONG)
    args = step.args()
    tree_attention(**args)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tree_attention(**args))
        graphs.append(graph)
    for i, lengths in enumerate(([2000, 700], [50, 90], [1333, 100])):
        args["lengths"].copy_(torch.tensor(lengths))
        if tree and i:
            args["mask"].copy_(~args["mask"])
        if i == 2:
            args["page_table"].copy_(args["page_table"].flip(0))
            args["lengths"].copy_(torch.tensor([600, 1900]))
        want = tree_attention(**args)
        for out in outs:
            out.fill_(math.nan)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert torch.isfinite(want).all() and all(torch.equal(out, want) for out in outs)


def test_a_long_prompt():
    """Blocks of rows over every length of the triangle, against float64 on the whole scores; two sequences share their first pages."""
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens, heads, head_dim, page, shared = 3000, 4, 128, 32, 1024
    lengths = [shared + tokens, shared + 700]
    need = [-(-n // page) for n in lengths]
    own = torch.randperm(sum(need), generator=g, device="cuda").int()
    table = torch.full((2, max(need)), -1, dtype=torch.int32, device="cuda")
    table[0, :need[0]], table[1, :need[1]] = own[:need[0]], own[need[0]:]
    table[1, :shared // page] = table[0, :shared // page]
    cache = [torch.randn(sum(need), page, 1, head_dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)]
    query = torch.randn(tokens + 700, heads, head_dim, generator=g, device="cuda").to(torch.bfloat16)
    starts = torch.tensor([0, tokens, tokens + 700], dtype=torch.int32, device="cuda")
    got = tree_attention(query, *cache, table, torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts)
    for b, length in enumerate(lengths):
        first, last = (0, tokens) if b == 0 else (tokens, tokens + 700)
        k, v = (c[table[b, :need[b]].long(), :, 0].reshape(-1, head_dim)[:length].double() for c in cache)
        sees = torch.ones(last - first, length, dtype=torch.bool, device="cuda").tril(shared)
        for h in range(heads):
            q = query[first:last, h].double()
            score = (q @ k.T) * head_dim ** -0.5
            # a score's error as in the oracle
            off = ((q.abs() @ k.abs().T) * head_dim ** -0.5).masked_fill(~sees, 0).amax(1) * (head_dim + 4) * 2.0 ** -24
            off = off + (score.abs().masked_fill(~sees, 0).amax(1) * 4 + 4) * 2.0 ** -23
            p = torch.softmax(score.masked_fill(~sees, -math.inf), 1)
            found = p @ v, p @ v.abs(), off, v.abs().amax(0).expand(last - first, -1)
            tol = oracle.attention_tolerance(found, torch.bfloat16, length)
            assert float(((got[first:last, h].double() - found[0]).abs() / tol).max()) <= 1.0


def test_starts_that_go_back_write_no_other_rows():
    """Starts have to rise; others give rows that mean nothing, but no row of no sequence is written and the next call is as it was."""
    step = Step([600] * 30, [2] * 30, 4, 2, 64, 16, extra=5)
    args = step.args()
    want = tree_attention(**args)
    out = torch.full(step.query.shape, 7.0, dtype=torch.bfloat16, device="cuda")
    back = torch.tensor([0 if i % 2 == 0 else 60 for i in range(31)], dtype=torch.int32, device="cuda")
    tree_attention(**{**args, "starts": back}, output=out)
    assert (out[60:] == 7.0).all()
    assert torch.equal(tree_attention(**args)[:60], want[:60])


def test_nothing_to_do():
    step = Step([5], [1], 4, 2, 64, 16, uniform=True)
    args = step.args()
    none = tree_attention(**{**args, "query": args["query"][:0]})
    assert none.shape == (0, 4, 64)
    no_seqs = {**args, "query": args["query"][:0], "page_table": args["page_table"][:0], "lengths": args["lengths"][:0]}
    assert tree_attention(**no_seqs).shape == (0, 4, 64)


def test_two_streams_at_once():
    steps = [Step([4000], [1], 8, 2, 128, 16, seed=s) for s in (1, 2)]
    args = [s.args() for s in steps]
    want = [tree_attention(**a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(tree_attention(**args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


def test_graphs_replayed_with_other_lengths():
    """A captured step follows what the lengths, the table and the cache hold at its replay; two graphs have workspaces of their own."""
    step = Step([3000, 900], [2, 2], 8, 2, 128, 16, seed=5)
    args = step.args()
    tree_attention(**args)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tree_attention(**args))
        graphs.append(graph)
    for lengths in ([3000, 900], [10, 2500], [2, 2], [1700, 3]):
        args["lengths"].copy_(torch.tensor([min(lengths[0], 3000), min(lengths[1], 900)]))
        want = tree_attention(**args)
        for out in outs:
            out.fill_(math.nan)
        streams = [torch.cuda.Stream() for _ in graphs]
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want) for out in outs)


@pytest.mark.parametrize("cache", [None, FP8])
def test_a_run_of_steps(cache):
    """Prompts, then drafted trees, then single tokens through append and attention, as they are used; the cache the oracle reads is what the
    append has written."""
    g = torch.Generator().manual_seed(11)
    heads, kv_heads, head_dim, page, seqs = 8, 2, 64, 16, 2
    pages = 20
    caches = [torch.full((pages, page, kv_heads, head_dim), math.nan).to(cache or torch.bfloat16).cuda() for _ in range(2)]
    table = torch.randperm(pages, generator=g)[:seqs * 6].view(seqs, 6).int()
    scales = [torch.tensor([0.02], device="cuda"), torch.tensor([0.015], device="cuda")] if cache else [None, None]
    frequencies, magnitude = rotary_frequencies(head_dim, 500000.0, {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32})
    held = [0, 0]
    for counts, tree in (([40, 23], False), ([5, 7], True), ([1, 1], False), ([3, 0], False)):
        total = sum(counts)
        rows = torch.randn(total, heads + 2 * kv_heads, head_dim, generator=g).to(torch.bfloat16).cuda()
        lengths = [h + n for h, n in zip(held, counts)]
        at = [(b, t) for b in range(seqs) for t in range(held[b], lengths[b])]
        slots = torch.tensor([int(table[b, t // page]) * page + t % page for b, t in at], device="cuda")
        positions = torch.tensor([t for _, t in at], device="cuda")
        query = append_kv(rows[:, heads:heads + kv_heads], rows[:, heads + kv_heads:], *caches, slots, positions, frequencies, magnitude=magnitude,
                          query=rows[:, :heads], key_scale=scales[0], value_scale=scales[1])
        mask = (torch.rand(total, max(counts), generator=g) < 0.5) if tree else None
        starts = torch.tensor([0, counts[0], total], dtype=torch.int32)
        got = tree_attention(query, *caches, table.cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda"), starts.cuda(),
                             None if mask is None else mask.cuda(), key_scale=scales[0], value_scale=scales[1])
        found = oracle.attention(query.cpu(), caches[0].cpu(), caches[1].cpu(), table, torch.tensor(lengths), starts, mask, head_dim ** -0.5,
                                 *[None if s is None else s.cpu() for s in scales])
        assert ((got.cpu().double() - found[0]).abs() <= oracle.attention_tolerance(found, torch.bfloat16, max(lengths))).all()
        held = lengths


def test_refused_on_the_device():
    step = Step([40], [2], 4, 2, 64, 16)
    args = step.args()
    with pytest.raises(RuntimeError, match="apart"):
        tree_attention(**args, output=args["query"])
    with pytest.raises(RuntimeError, match="aligned"):
        odd = torch.zeros(2 * 4 * 64 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 4, 64)
        tree_attention(**{**args, "query": odd})
    with pytest.raises(AssertionError, match="lengths"):
        tree_attention(**{**args, "lengths": args["lengths"].cpu()})


def test_whole_calls_and_general_ones_give_the_same_bits(monkeypatch):
    from hf_rocm_kernels.operators.tree_attention import wrapped
    step = Step([1000, 45], [4, 3], 8, 2, 64, 16, tree="full", seed=12)
    args = step.args()
    scale = torch.tensor([0.01], device="cuda")
    calls = lambda: [tree_attention(**args), tree_attention(**args, scale=0.3), tree_attention(**args, out_scale=scale).view(torch.uint8)]
    got = calls()
    monkeypatch.setattr(wrapped, "_tree_attention_new", lambda *args: None)
    assert all(torch.equal(a, b) for a, b in zip(got, calls()))


def small_weights(far, length, page, tokens, heads, cache, places=0):
    """(arguments, head groups' far, first row's place): queries and keys whose scores are in powers of two: `far` for the first token, 0 for the others, the first token's
    value is 0 and the others' 448.  The step is a chain."""
    pages = -(-length // page)
    key, value = torch.zeros(pages, page, 1, 16), torch.full((pages, page, 1, 16), 448.0)
    key[0, 0, 0, :2] = torch.tensor([far // 8 * 8, far % 8]) if cache != FP8 else torch.tensor([8.0, 8.0])
    value[0, 0] = 0.0
    query = torch.zeros(tokens, heads, 16)
    query[..., :2] = 1.0 if cache != FP8 else far / 16
    query = query.to(torch.float16)
    columns = max(pages, places // page)
    table = torch.zeros(1, columns, dtype=torch.int32)
    table[0, :pages] = torch.arange(pages)
    far = (query[0, 0].double() * key[0, 0, 0].to(cache).double()).sum()
    return (query, key.to(cache), value.to(cache), table, torch.tensor([length], dtype=torch.int32), None, None, math.log(2.0)), far, length - tokens


def check_small_weights(got, far, front):
    """A weight in fp16 is off by half a step of itself and by 2^-25 where the largest is at least 2^7, in the sum above and in the one below the line; the scale ln 2 is a
    float, as are the score and the exponential (2^-24 of `far` each, and 2^-22): then one rounding."""
    weight = 2.0 ** -float(far)
    tail = torch.arange(front, front + got.size(0), dtype=torch.float64)  # tokens behind the first that a row sees
    want = 448.0 * tail * weight / (1.0 + tail * weight)
    off = 2 * (2.0 ** -11 + 2.0 ** -32 / weight + 4 * float(far) * 2.0 ** -24 + 2.0 ** -22) + 2 * float(tail.max()) * 2.0 ** -24
    tolerance = want * (off * (1 + 2.0 ** -8) + 2.0 ** -11) + oracle.smallest_step(torch.float16)
    assert ((got.cpu().double() - want[:, None, None]).abs() <= tolerance[:, None, None]).all()


@pytest.mark.parametrize("far", [21.5, 23.5, 24.6, 25.0, 28.0])
@pytest.mark.parametrize("tokens,heads,cache", [(1, 2, torch.float16), (3, 8, FP8), (70, 8, torch.float16), (20, 8, FP8)])
def test_many_small_weights_beside_a_large_one_in_fp16(far, tokens, heads, cache):
    """Rows far longer than fp16 has steps below the largest weight: a first token with a large score and a value of zero, and a flat tail."""
    args, far, front = small_weights(far, 131072, 64, tokens, heads, cache)
    check_small_weights(tree_attention(*[t.cuda() if torch.is_tensor(t) else t for t in args]), far, front)


def minus_infinities(dtype, counts, front, heads, head_dim, tree, places):
    """The first sequence's keys are minus infinity, its queries positive: rows of it that see something have no softmax, and rows that see nothing are zero.  The
    second's are so up to its step, which counts for nothing beside a finite score."""
    step = Step([n + front for n in counts], counts, heads, 2, head_dim, 16, dtype, tree="full" if tree else None, seed=7, places=places)
    step.query = step.query.abs() + 0.25
    for b, end in ((0, step.lengths[0]), (1, front)):
        for t in range(end):
            step.key[int(step.table[b, t // 16]), t % 16] = -math.inf
    if tree:
        step.mask[1] = False
    return step


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("counts,front,heads,head_dim,places", [([1, 1], 40, 4, 64, 0), ([3, 2], 0, 4, 128, 0), ([5, 9], 700, 8, 256, 0), ([40, 36], 0, 8, 64, LONG),
                                                                ([40, 70], 300, 8, 128, LONG), ([33, 40], 20, 4, 256, LONG)])
@pytest.mark.parametrize("tree", [False, True])
def test_scores_of_minus_infinity(dtype, counts, front, heads, head_dim, places, tree):
    step = minus_infinities(dtype, counts, front, heads, head_dim, tree, places)
    step.check(tree_attention(**step.args()))


def test_more_rows_than_a_launch_has_threads():
    """A last row of 2^27, whose parts are joined: more groups of 32 lanes than 32 bits count threads."""
    tokens, heads, head_dim, page, long = (1 << 21) + 1, 64, 144, 4096, 1 << 22
    g = torch.Generator(device="cuda").manual_seed(2)
    key, value = (torch.randn(1, page, heads, head_dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2))
    query = torch.randn(1, heads, head_dim, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.zeros(2, long // page, dtype=torch.int32, device="cuda")  # one page, over and over
    starts = torch.tensor([0, tokens - 1, tokens], dtype=torch.int32, device="cuda")
    out = torch.full((tokens, heads, head_dim), 7.0, dtype=torch.bfloat16, device="cuda")
    tree_attention(query.expand(tokens, heads, head_dim), key, value, table, torch.tensor([8, long], dtype=torch.int32, device="cuda"), starts, output=out)
    # the page's weights 1024 times over; products of 16 tokens are added one after the other, 2^18 of them at most
    q, k, v = query[0].cpu().double(), key[0].cpu().double().transpose(0, 1), value[0].cpu().double().transpose(0, 1)
    score = torch.matmul(k, q[:, :, None])[..., 0] * head_dim ** -0.5
    off = torch.matmul(k.abs(), q.abs()[:, :, None])[..., 0].amax(1) * head_dim ** -0.5 * (head_dim + 4) * 2.0 ** -24 + (score.abs().amax(1) * 4 + 4) * 2.0 ** -23
    p = torch.softmax(score, 1)[:, None]
    found = torch.matmul(p, v)[:, 0], torch.matmul(p, v.abs())[:, 0], off, v.abs().amax(1)
    assert ((out[-1].cpu().double() - found[0]).abs() <= oracle.attention_tolerance(found, torch.bfloat16, long // 16)).all()
    assert not out[:tokens - 9].any()  # rows that see nothing


@pytest.mark.parametrize("places", [0, LONG])
def test_a_result_in_fp8_keeps_nan(places):
    step = minus_infinities(torch.bfloat16, [40, 40], 0, 8, 64, False, places)
    got = tree_attention(**step.args(), out_scale=torch.tensor([0.01], device="cuda")).float()
    assert torch.isnan(got[:40]).all() and torch.isfinite(got[40:]).all()
