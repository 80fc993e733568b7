"""Drafted trees over blocks of KV memory: tree_attn, block_tables and tree_commit against plain implementations in 64 bits
(attention) and in Python integers, at the sizes, masks, strides and cache contents where they can go wrong."""

import functools
import math
import threading

import pytest
import torch

from quic_cu_b200 import kernels as K

pytestmark = pytest.mark.gpu
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}  # a rounding's relative error at most


@pytest.fixture(params=["mma", "tensor"])
def form(request):
    """Each of the attention's two forms, whichever the sizes would choose."""
    K.lib().quic_set_tree_attn_tensor(int(request.param == "tensor"))
    yield request.param
    K.lib().quic_set_tree_attn_tensor(-1)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _random_parents(n, seed):
    g = torch.Generator().manual_seed(seed)
    return [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=g)) for i in range(1, n)]


def _ancestors(parents, i):
    seen = set()
    while i >= 0:
        seen.add(i)
        i = parents[i]
    return seen


def _pack(sees, words):
    """Bit masks, 32 to a word, of lists of sets."""
    rows = []
    for s in sees:
        w = [sum(1 << (j - 32 * k) for j in s if 32 * k <= j < 32 * k + 32) for k in range(words)]
        rows.append([x - 2 ** 32 if x >= 2 ** 31 else x for x in w])
    return torch.tensor(rows, dtype=torch.int32, device="cuda").view(len(sees), words)


class Case:
    """Requests with a blocked cache whose blocks lie in any order, and what every row sees (None: a chain)."""

    def __init__(self, lengths, new, block, heads=14, kv_heads=2, dim=64, dtype=torch.float16, tree=True, seed=0, spare=2,
                 scale=1.0, skip_rows=0):
        self.lengths, self.new, self.block, self.dim, self.heads, self.kv_heads = lengths, new, block, dim, heads, kv_heads
        g = _gen(seed)
        counts = [max(1, -(-(n + m) // block)) for n, m in zip(lengths, new)]
        ids = torch.randperm(sum(counts) + spare, generator=torch.Generator().manual_seed(seed)).tolist()
        self.tables = torch.full((len(new), max(counts)), -1, dtype=torch.int32)
        for b, c in enumerate(counts):
            self.tables[b, :c] = torch.tensor([ids.pop() for _ in range(c)], dtype=torch.int32)
        self.tables = self.tables.cuda()
        shape = (sum(counts) + spare, kv_heads, block, dim)
        self.k, self.v = (torch.randn(shape, device="cuda", generator=g).to(dtype) for _ in range(2))
        self.starts = [skip_rows]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.q = (scale * torch.randn(self.starts[-1], heads, dim, device="cuda", generator=g)).to(dtype)
        self.words = max(1, -(-max(new, default=1) // 32))
        self.trees = [_random_parents(n, seed + b) if n else [] for b, n in enumerate(new)]
        self.sees = [[_ancestors(t, i) if tree else set(range(i + 1)) for i in range(len(t))] for t in self.trees]
        self.mask = None
        if tree:
            self.set_mask()

    def set_mask(self):
        rows = [set()] * self.starts[0] + [s for t in self.sees for s in t]
        self.mask = _pack(rows, self.words)

    def place(self, b, p):
        return int(self.tables[b, p // self.block]), p % self.block

    def clear_unused(self, value=float("nan")):
        """What no position of any request uses holds `value`."""
        for t in (self.k, self.v):
            used = torch.zeros(t.shape[0], self.block, dtype=torch.bool, device="cuda")
            for b in range(len(self.new)):
                for p in range(self.lengths[b] + self.new[b]):
                    used[self.place(b, p)] = True
            t.masked_fill_(~used[:, None, :, None], value)

    def call(self, **more):
        i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
        args = dict(mask=self.mask, max_new=max(max(self.new), 1), max_len=max(self.lengths))
        args.update(more)
        return K.tree_attn(self.q, self.k, self.v, self.tables, i32(self.lengths), i32(self.starts), **args)

    def want(self, softmax_scale=None):
        """In 64 bits, and the sum of |p v| that the roundings scale with."""
        scale = softmax_scale or self.dim ** -0.5
        out = torch.zeros(self.q.shape, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            total = self.lengths[b] + n
            ids = self.tables[b, :-(-total // self.block)].long()
            for h in range(self.kv_heads):
                k, v = (t[ids, h].reshape(-1, self.dim)[:total].double() for t in (self.k, self.v))
                for i in range(n):
                    at = torch.tensor(list(range(self.lengths[b])) + [self.lengths[b] + j for j in sorted(self.sees[b][i]) if j < n],
                                      device="cuda", dtype=torch.long)
                    if at.numel() == 0:
                        continue
                    row = self.starts[b] + i
                    q = self.q[row, h * group:(h + 1) * group].double()
                    p = torch.softmax(q @ k[at].T * scale, -1)
                    out[row, h * group:(h + 1) * group] = p @ v[at]
                    size[row, h * group:(h + 1) * group] = p @ v[at].abs()
        return out, size

    def check(self, got, softmax_scale=None):
        """Roundings: each weight once to the type, the sum of the rounded weights (off by at most as much), the result once:
        3 half steps of sum |p v|; fp32 sums and exponentials far below: 0.2.  fp16 weights are held as 2^7 p by a reference that
        is not above the largest, so those below 2^-21 (subnormal: half a step is 2^-25) are off by 2^-32 of the largest, with
        |v| < 8; fp16 results below 2^-14 by 2^-25."""
        want, size = self.want(softmax_scale)
        half = HALF[self.q.dtype]
        limit = (3.2 * half) * size + 2.0 ** -24
        if self.q.dtype is torch.float16:
            limit = limit + (max(self.lengths) + max(self.new)) * 2.0 ** -32 * 8
        rows = slice(self.starts[0], self.starts[-1])
        worst = ((got.double() - want).abs() / limit)[rows].max().item() if self.starts[-1] > self.starts[0] else 0.0
        assert worst <= 1.0, worst


TYPES = [torch.float16, torch.bfloat16]
LAYOUTS = [(14, 2, 64), (32, 8, 128), (8, 8, 64), (16, 1, 128), (3, 1, 64)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("tree", [True, False])
def test_attention_of_ragged_requests(form, dtype, layout, tree):
    heads, kv_heads, dim = layout
    case = Case([0, 1, 63, 64, 65, 500, 1023], [1, 7, 0, 33, 2, 16, 5], 16, heads, kv_heads, dim, dtype, tree, seed=heads)
    case.clear_unused()
    case.check(case.call())


@pytest.mark.parametrize("block", [1, 5, 8, 16, 24, 64, 100, 700, 1024])
@pytest.mark.parametrize("nodes", [1, 3, 40])
def test_blocks_of_any_size(form, block, nodes):
    case = Case([333, 17, 600], [nodes, 1, nodes], block, seed=block + nodes)
    case.clear_unused()
    case.check(case.call())


@pytest.mark.parametrize("lengths,new", [([0], [1]), ([1], [1]), ([31], [1]), ([32], [1]), ([4000], [1]), ([4001], [64]), ([0], [64]),
                                         ([20000], [48]), ([9000], [200]), ([0, 0], [130, 1]), ([2000] * 40, [8] * 40)])
@pytest.mark.parametrize("dtype", TYPES)
def test_lengths(form, lengths, new, dtype):
    case = Case(lengths, new, 32, dtype=dtype, seed=len(new))
    case.clear_unused()
    case.check(case.call())


def test_a_row_that_sees_nothing_is_zero(form):
    case = Case([0, 0, 40], [5, 3, 4], 16, seed=3)
    case.sees[0] = [{0}, set(), {1, 4}, {0, 1, 2, 3, 4}, {7, 40}]  # nodes that are not there, and later ones
    case.sees[2] = [set()] * 4
    case.words = 2
    case.set_mask()
    case.clear_unused()
    got = case.call()
    assert torch.count_nonzero(got[1]) == 0 and torch.count_nonzero(got[4]) == 0
    case.check(got)


@pytest.mark.parametrize("layout", LAYOUTS[:2])
@pytest.mark.parametrize("nodes", [2, 9, 50])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
def test_what_a_row_does_not_see_does_not_reach_it(form, layout, nodes, value):
    """The last node of each tree (which no other sees) holds infinities or NaN in K and V: only its own row shows it."""
    heads, kv_heads, dim = layout
    case = Case([70, 0, 301], [nodes] * 3, 16, heads, kv_heads, dim, seed=nodes)
    clean = case.call().clone()
    for b in range(3):
        for s in case.sees[b][:-1]:
            assert nodes - 1 not in s
        block, off = case.place(b, case.lengths[b] + nodes - 1)
        case.v[block, :, off] = value
    got = case.call()
    for b in range(3):
        last = case.starts[b + 1] - 1
        assert torch.equal(got[case.starts[b]:last], clean[case.starts[b]:last])
        row = got[last].float()
        assert torch.isnan(row).all() if math.isnan(value) else (row == value).all()
    for b in range(3):
        block, off = case.place(b, case.lengths[b] + nodes - 1)
        case.k[block, :, off] = float("nan")
    got = case.call()
    for b in range(3):
        last = case.starts[b + 1] - 1
        assert torch.equal(got[case.starts[b]:last], clean[case.starts[b]:last])
        assert torch.isnan(got[last].float()).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", LAYOUTS[:2])
@pytest.mark.parametrize("block", [5, 8, 24, 64])
@pytest.mark.parametrize("nodes,tree", [(3, True), (3, False), (40, True), (40, False)])
def test_a_node_that_is_not_finite_reaches_the_rows_that_see_it(form, dtype, layout, block, nodes, tree):
    """One value of one node's V is an infinity or NaN: the results of the rows that see the node show it there, and nothing else
    changes; so it is for the last node, which without masks only its own row sees."""
    heads, kv_heads, dim = layout
    case = Case([70, 0, 301], [nodes, 2, nodes - 1], block, heads, kv_heads, dim, dtype, tree, seed=nodes + block)
    clean, group = case.call().clone(), heads // kv_heads
    for value, node in ((float("nan"), 1), (float("inf"), nodes // 2), (float("-inf"), nodes - 1)):
        v = case.v.clone()
        places, odd = [], torch.zeros_like(clean, dtype=torch.bool)
        for b in range(3):
            at = min(node, case.new[b] - 1)
            place, off = case.place(b, case.lengths[b] + at)
            case.v[place, 1, off, dim - 3] = value
            for i, sees in enumerate(case.sees[b]):
                if at in sees:
                    odd[case.starts[b] + i, group:2 * group, dim - 3] = True
        got = case.call()
        assert torch.equal(got[~odd], clean[~odd]) and odd.any() and not odd.all(0).any()
        assert torch.isnan(got[odd]).all() if math.isnan(value) else (got[odd] == value).all()
        case.v = v


def test_a_nan_score_reaches_its_rows(form):
    case = Case([3], [2], 16, seed=1)
    case.k[case.place(0, 1)[0], 0, 1] = float("nan")
    got = case.call()
    assert torch.isnan(got[:, :7].float()).all() and torch.isfinite(got[:, 7:].float()).all()


@pytest.mark.parametrize("key", range(0, 70, 3))
def test_a_nan_score_of_any_key_reaches_its_rows(key):
    """Whichever way the tcgen05 form takes for the key's exponential; unseen keys and scores far below stay without a trace."""
    K.lib().quic_set_tree_attn_tensor(1)
    try:
        case = Case([70], [3], 16, tree=False, seed=key)
        case.k[case.place(0, key)[0], 0, case.place(0, key)[1], 5] = float("nan")
        got = case.call()
        assert torch.isnan(got[:, :7]).all() and not torch.isnan(got[:, 7:]).any()
        case = Case([70], [3], 16, tree=False, seed=key, dtype=torch.bfloat16)
        block, at = case.place(0, key)
        case.q[...] = 1.0
        case.k[...] = 30.0
        case.k[block, :, at] = -30.0  # 2^-690 beside the others'
        case.v[block, :, at] = 3e38
        assert (case.call().abs() < 8).all()
    finally:
        K.lib().quic_set_tree_attn_tensor(-1)


def test_scores_of_the_lowest_value(form):
    """Keys that push a score to the type's end in either direction: the softmax stays finite."""
    case = Case([100], [6], 16, seed=2)
    case.q.fill_(255.0)
    for p in range(106):
        block, off = case.place(0, p)
        case.k[block, :, off] = -255.0 if p % 3 else 255.0
    got = case.call()
    assert torch.isfinite(got.float()).all()
    case.check(got)


def test_rows_outside_the_requests_stay_as_they_were(form):
    case = Case([30, 50], [4, 3], 16, seed=5, skip_rows=2)
    case.q = torch.cat([case.q, case.q[:5]])
    case.mask = torch.cat([case.mask, case.mask[:5]])
    out = torch.full_like(case.q, 7.0)
    assert case.call(out=out) is out
    assert (out[:2] == 7).all() and (out[9:] == 7).all()
    want, _ = Case.want(case)
    assert (out[2:9].double() - want[2:9]).abs().max() < 1e-2


@pytest.mark.parametrize("nodes", [1, 20])
def test_strides(form, nodes):
    """Heads before rows in q, tokens before heads in the cache, K and V side by side, table rows and mask rows apart."""
    case = Case([200, 90], [nodes, nodes], 16, seed=nodes)
    want = case.call()
    case.q = case.q.transpose(0, 1).contiguous().transpose(0, 1)
    both = torch.stack([case.k.transpose(1, 2), case.v.transpose(1, 2)], 2).contiguous()  # [blocks, block, 2, heads, dim]
    case.k, case.v = both[:, :, 0].transpose(1, 2), both[:, :, 1].transpose(1, 2)
    case.tables = torch.nn.functional.pad(case.tables, (0, 3))[:, :case.tables.shape[1]]
    case.mask = torch.nn.functional.pad(case.mask, (0, 2))[:, :case.mask.shape[1]]
    assert torch.equal(case.call(), want)
    case.k = both[:, :, 0].contiguous().transpose(1, 2)  # K and V of different strides
    assert torch.equal(case.call(), want)


def test_shared_keys(form):
    """Two requests over the same blocks, one KV head for all heads (stride 0)."""
    case = Case([130, 130], [3, 3], 16, seed=9)
    case.tables[1] = case.tables[0]
    case.k, case.v = case.k[:, :1].expand(-1, 2, -1, -1), case.v[:, :1].expand(-1, 2, -1, -1)
    case.check(case.call())


@pytest.mark.parametrize("nodes", [1, 30])
def test_bad_blocks_are_seen_by_nobody(form, nodes):
    case = Case([170], [nodes], 16, seed=nodes)
    case.check(case.call())
    whole = case.k.shape[0]
    keep = [p for p in range(170 + nodes) if not (16 <= p < 32 or 96 <= p < 112)]
    case.tables[0, 1], case.tables[0, 6] = -5, whole
    got = case.call()
    flat = [case.place(0, p) for p in keep]
    k = torch.stack([case.k[b, :, o] for b, o in flat], 1).double()  # [heads, keys, dim]
    v = torch.stack([case.v[b, :, o] for b, o in flat], 1).double()
    for i in range(nodes):
        at = torch.tensor([j for j, p in enumerate(keep) if p < 170 or p - 170 in case.sees[0][i]], device="cuda")
        q = case.q[i].double().view(2, 7, 64)
        want = torch.softmax(q @ k[:, at].transpose(1, 2) / 8, -1) @ v[:, at]
        assert (got[i].double().view(2, 7, 64) - want).abs().max() < 4e-3


def test_tables_shorter_than_the_lengths(form):
    """Positions that the table has no entry for are seen by nobody; nothing is read there."""
    case = Case([64], [4], 16, seed=4)
    case.tables = case.tables[:, :4].contiguous()
    got = case.call()
    case.sees[0] = [set()] * 4
    case.check(got)


@pytest.mark.parametrize("bounds", [dict(max_new=None, max_len=None), dict(max_len=0), dict(max_new=100), dict(max_len=10 ** 6)])
def test_bounds_only_plan(form, bounds):
    case = Case([700, 5], [9, 1], 16, seed=6)
    case.check(case.call(**bounds))


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("most", [1, 5, 33])
@pytest.mark.parametrize("dtype,layout", [(torch.float16, (14, 2, 64)), (torch.bfloat16, (32, 8, 128))])
def test_rows_beyond_the_bound_stay_unwritten(form, tree, most, dtype, layout):
    """max_new below the rows of some requests: the rows up to it are right, the others of the request as they were."""
    case = Case([300, 0, 41, 2000], [40, 3, 6, 34], 16, *layout, dtype=dtype, tree=tree, seed=most)
    case.clear_unused()
    out = torch.full_like(case.q, 7.0)
    assert case.call(out=out, max_new=most) is out
    want, size = case.want()
    limit = 3.2 * HALF[dtype] * size + 2.0 ** -24 + (2040 * 2.0 ** -32 * 8 if dtype is torch.float16 else 0.0)  # (as in Case.check)
    for b, n in enumerate(case.new):
        s, e = case.starts[b], case.starts[b] + min(n, most)
        assert ((out[s:e].double() - want[s:e]).abs() <= limit[s:e]).all()
        assert (out[e:case.starts[b + 1]] == 7).all()


def test_scale(form):
    case = Case([90], [5], 16, seed=8)
    case.check(case.call(softmax_scale=0.31), 0.31)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("longest,nodes", [(70, 1), (200, 3), (460, 1), (511, 2), (2040, 1), (2100, 4)])
def test_requests_of_any_length_beside_a_long_one(form, dim, longest, nodes):
    """Parts of a request by those of the longest: none, one, fewer, all."""
    lengths = [longest, 0, 1, 62, 63, 64, longest // 2, longest - 1]
    case = Case(lengths, [nodes, 1, 0, 1, nodes, 1, nodes, 2], 16, 4, 2, dim, seed=longest)
    case.check(case.call())


@pytest.mark.parametrize("tree", [True, False])
@pytest.mark.parametrize("requests,nodes,layout,dtype", [(20, 28, (32, 8, 128), torch.float16), (40, 17, (14, 2, 64), torch.bfloat16),
                                                         (64, 16, (32, 8, 128), torch.bfloat16)])
def test_short_requests_of_many_rows(form, requests, nodes, layout, dtype, tree):
    """More row tiles than CTAs run at once, few keys: a warp has rows of its own."""
    lengths, new = [(5 * b) % 16 for b in range(requests)], [nodes - b % 3 if b % 7 else b % 2 for b in range(requests)]
    case = Case(lengths, new, 16, *layout, dtype=dtype, tree=tree, seed=nodes)
    case.clear_unused()
    case.check(case.call())


@pytest.mark.parametrize("lengths,new", [([40], [3]), ([900, 20], [4, 9]), ([3000] * 3, [40] * 3)])
def test_results_in_the_place_of_the_queries(form, lengths, new):
    case = Case(lengths, new, 16, seed=4)
    want, q = case.call(), case.q.clone()
    assert case.call(out=case.q) is case.q and torch.equal(case.q, want)
    case.q = q
    case.check(want)


def test_offsets_beyond_32_bits(form):
    """Blocks that begin beyond element 2^31 of planes of 4.3 GB each."""
    block, blocks = 4096, 4100
    planes = torch.zeros(2, blocks * block * 2 * 64 + 8, dtype=torch.float16, device="cuda")
    case = Case([5000], [3], block, seed=7)
    k, v = (p[:blocks * block * 128].view(blocks, 2, block, 64) for p in planes)
    for i, far in enumerate((4097, 4099)):
        k[far], v[far] = case.k[case.tables[0, i]], case.v[case.tables[0, i]]
    want = case.call()
    case.k, case.v, case.tables = k, v, torch.tensor([[4097, 4099]], dtype=torch.int32, device="cuda")
    assert torch.equal(case.call(), want)


def test_another_stream_and_graphs(form):
    """On a side stream, and in two graphs that are replayed in turn with an eager call between."""
    cases = [Case([3000], [20], 16, seed=1), Case([9000, 10], [1, 4], 32, seed=2)]
    want = [c.call().clone() for c in cases]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(cases[0].call(), want[0])
    torch.cuda.current_stream().wait_stream(side)
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    graphs, outs, inputs = [], [], [(i32(c.lengths), i32(c.starts)) for c in cases]
    for c, (lengths, starts) in zip(cases, inputs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(K.tree_attn(c.q, c.k, c.v, c.tables, lengths, starts, mask=c.mask, max_new=max(c.new), max_len=max(c.lengths)))
        graphs.append(g)
    for _ in range(3):
        for g in graphs:
            g.replay()
        assert torch.equal(cases[0].call(), want[0])
        for o, w in zip(outs, want):
            assert torch.equal(o, w)
            o.zero_()


def test_two_graphs_at_once(form):
    """Captured on a stream that has run the operator before, replayed on two streams at once beside eager calls on the first."""
    cases = [Case([6000, 9000], [20, 3], 16, seed=s) for s in (1, 2)]
    want = [c.call().clone() for c in cases]
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    lengths, starts = i32(cases[0].lengths), i32(cases[0].starts)
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []

    def call(c):
        return K.tree_attn(c.q, c.k, c.v, c.tables, lengths, starts, mask=c.mask, max_new=20, max_len=9000)

    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        call(cases[0])
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            outs.append(call(c))
        graphs.append(g)
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(streams[0]):
            eager = call(cases[1])
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[1])


def test_same_result_every_time(form):
    case = Case([2500] * 3, [30, 2, 17], 16, seed=12)
    want = case.call()
    for _ in range(5):
        assert torch.equal(case.call(), want)


def test_the_rule_between_the_forms():
    """Calls on both sides of the rule, in either form and by the rule: one result up to the roundings."""
    for lengths, new, layout in (([1600] * 40, [8] * 40, (14, 2, 64)), ([3000], [48], (14, 2, 64)), ([5000] * 9, [2] * 9, (16, 1, 128))):
        case = Case(lengths, new, 16, *layout, seed=len(new))
        got = []
        for mode in (0, 1, -1):
            K.lib().quic_set_tree_attn_tensor(mode)
            got.append(case.call())
        K.lib().quic_set_tree_attn_tensor(-1)
        assert torch.equal(got[2], got[0]) or torch.equal(got[2], got[1])
        case.check(got[0])
        case.check(got[1])


def test_many_requests(form):
    """More requests than threads look at, empty ones among them, and more rows per request than one tile of any form has."""
    lengths = [(7 * b) % 90 for b in range(1500)]
    new = [(b * b) % 4 for b in range(1500)]
    lengths[700], new[700] = 300, 90
    case = Case(lengths, new, 8, 8, 8, 64, seed=2)
    case.check(case.call())


@pytest.mark.parametrize("layout", [(14, 2, 64), (32, 8, 128)])
def test_waits_that_give_up(layout):
    """The tcgen05 form's bounded waits: K and V that come late change nothing; a tile that never comes sets the error word, and
    the next call is right."""
    lib = K.lib()
    lib.quic_set_tree_attn_tensor(1)
    try:
        for nodes in (3, 40):
            case = Case([2000, 900], [nodes, nodes], 16, *layout, seed=nodes)
            want = case.call().clone()
            assert lib.quic_w4a16_tensor_status() == 0
            for limit, skip, fails in ((1500, -600, False), (1500, 0, True), (1500, 1, True)):
                lib.quic_w4a16_tensor_test_hook(limit, skip)
                try:
                    got = case.call().clone()
                finally:
                    lib.quic_w4a16_tensor_test_hook(0, -1)
                assert (lib.quic_w4a16_tensor_status() != 0) == fails
                assert fails or torch.equal(got, want)
                assert torch.equal(case.call(), want)
                assert lib.quic_w4a16_tensor_status() == 0
    finally:
        lib.quic_set_tree_attn_tensor(-1)


@pytest.mark.parametrize("layout", [(14, 2, 64), (32, 8, 128)])
def test_an_issuer_that_is_late_where_it_has_no_step(layout):
    """Requests of one key tile each, several to a CTA of the tcgen05 form: the second stream has nothing to do, and its issuer comes
    two tiles' time late to every one of them."""
    lib = K.lib()
    heads, kv_heads, dim = layout
    requests = 1200 // kv_heads
    case = Case([(7 * b) % 60 for b in range(requests)], [1 + b % 3 for b in range(requests)], 16, heads, kv_heads, dim, seed=dim)
    lib.quic_set_tree_attn_tensor(1)
    try:
        want = case.call().clone()
        for late in (-200, -40):
            lib.quic_w4a16_tensor_test_hook(50000, late)
            try:
                got = case.call().clone()
            finally:
                lib.quic_w4a16_tensor_test_hook(0, -1)
            assert lib.quic_w4a16_tensor_status() == 0 and torch.equal(got, want)
        case.check(want)
    finally:
        lib.quic_set_tree_attn_tensor(-1)


@pytest.mark.parametrize("lengths,new", [([3000, 900], [40, 9]), ([8000], [3])])
def test_two_threads_on_one_stream(form, lengths, new):
    """A call is several launches, and those of three threads interleave: each has scratch memory of its own."""
    cases = [Case(lengths, new, 16, seed=s) for s in range(3)]
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    more = [(i32(c.lengths), i32(c.starts)) for c in cases]
    want, got, start = [c.call() for c in cases], [[] for _ in cases], threading.Barrier(3)

    def work(i):
        c = cases[i]
        start.wait()
        for _ in range(200):
            got[i].append(K.tree_attn(c.q, c.k, c.v, c.tables, *more[i], mask=c.mask, max_new=max(new), max_len=max(lengths)))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert len(outs) == 200 and all(torch.equal(o, w) for o in outs)


# ---- block_tables ----------------------------------------------------------------------------
class Pool:
    """block_tables in Python integers."""

    def __init__(self, requests, width, n_blocks, block):
        self.block, self.n, self.width = block, n_blocks, width
        self.tables = [[0] * width for _ in range(requests)]
        self.held, self.free = [0] * requests, list(range(n_blocks))

    def step(self, lengths, new, max_rows, parents=None, words=0):
        take = [max(n, 0) for n in new]
        want = [-(-(l + n) // self.block) for l, n in zip(lengths, take)]
        need = [max(0, w - h) if n else 0 for w, h, n in zip(want, self.held, take)]
        status = 0
        if any(n and w > self.width for n, w in zip(take, want)):
            status = -1
        elif sum(take) > max_rows or (parents is not None and (sum(take) > len(parents) or any(n > 32 * words for n in take))):
            status = -2
        elif sum(need) > len(self.free):
            status = sum(need) - len(self.free)
        if status:
            take, need = [0] * len(new), [0] * len(new)
        for b, k in enumerate(need):
            for _ in range(k):
                self.tables[b][self.held[b]] = self.free.pop(0)
                self.held[b] += 1
        for b, n in enumerate(new):
            if n < 0:
                self.free += self.tables[b][:self.held[b]]
                self.held[b] = 0
        starts = [0]
        slots, positions, masks = [], [], []
        for b, n in enumerate(take):
            starts.append(starts[-1] + n)
            for i in range(n):
                p = lengths[b] + i
                slots.append(self.tables[b][p // self.block] * self.block + p % self.block)
                seen = {i}
                if parents is not None:
                    node = i
                    while 0 <= parents[starts[b] + node] < node:
                        node = parents[starts[b] + node]
                        seen.add(node)
                    masks.append(seen)
                positions.append(lengths[b] + (len(seen) - 1 if parents is not None else i))
        rest = max_rows - len(slots)
        return status, starts, slots + [-1] * rest, positions + [0] * rest, masks + [set()] * rest


@pytest.mark.parametrize("requests,block,n_blocks,most,tree", [(1, 16, 4, 3, False), (5, 16, 40, 20, True), (64, 16, 300, 33, True),
                                                               (300, 7, 2000, 40, False), (257, 32, 900, 64, True), (4096, 16, 9000, 9, False)])
def test_tables_over_many_steps(requests, block, n_blocks, most, tree):
    """Requests come, grow and end; now and then the pool runs out, and nothing happens but a status."""
    width = 12
    model = Pool(requests, width, n_blocks, block)
    tables = torch.zeros(requests, width + 3, dtype=torch.int32, device="cuda")[:, :width]
    held = torch.zeros(requests, dtype=torch.int32, device="cuda")
    pool = K.block_pool(n_blocks, "cuda")
    g = torch.Generator().manual_seed(requests)
    lengths, seen = [0] * requests, set()
    for step in range(12):
        new = torch.randint(-2, most + 1, (requests,), generator=g).tolist()
        if step % 4 == 2:  # few requests at once
            new = [n if b % 5 == 0 else 0 for b, n in enumerate(new)]
        lengths = [0 if h == 0 else l for l, h in zip(lengths, model.held)]
        max_rows = sum(max(n, 0) for n in new) + (5 if step != 7 else -1)
        max_rows = max(max_rows, 0)
        parents = None
        if tree:
            parents = [int(x) for x in torch.randint(-1, most, (max(max_rows - 3 * (step % 3), 0),), generator=g)]
        i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
        got = K.block_tables(tables, held, pool, i32(lengths), i32(new), block, max_rows,
                             parents=None if parents is None else i32(parents), max_new=most)
        status, starts, slots, positions, masks = model.step(lengths, new, max_rows, parents, -(-most // 32))
        assert int(pool[3]) == status and int(pool[2]) == 0
        seen.add(status > 0)
        assert got[0].tolist() == starts and got[1].tolist() == slots and got[2].tolist() == positions
        assert got[1].dtype is torch.int64
        if parents is not None and max_rows:
            assert torch.equal(got[3], _pack(masks, -(-most // 32)))
        assert held.tolist() == model.held
        for b in range(requests):
            assert tables[b, :model.held[b]].tolist() == model.tables[b][:model.held[b]]
        head, count = int(pool[0]), int(pool[1])
        assert [int(pool[4 + (head + i) % n_blocks]) for i in range(count)] == model.free if n_blocks < 1000 else count == len(model.free)
        if status == 0:  # what is kept of the rows
            lengths = [0 if n < 0 else l + (n + 1) // 2 for l, n in zip(lengths, new)]


def test_tables_in_a_graph_and_without_a_pool():
    """Replayed, the call goes on from the state that it left; slots as blocks need no pool."""
    tables = torch.tensor([[3], [1], [2]], dtype=torch.int32, device="cuda")
    held = torch.ones(3, dtype=torch.int32, device="cuda")
    pool = K.block_pool(0, "cuda")
    lengths = torch.tensor([10, 0, 99], dtype=torch.int32, device="cuda")
    new = torch.tensor([2, 3, 1], dtype=torch.int32, device="cuda")
    K.block_tables(tables, held, pool, lengths, new, 100, 8)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        start, slots, positions, mask = K.block_tables(tables, held, pool, lengths, new, 100, 8)
    for _ in range(2):
        graph.replay()
        assert start.tolist() == [0, 2, 5, 6] and mask is None
        assert slots.tolist() == [310, 311, 100, 101, 102, 299, -1, -1] and positions.tolist() == [10, 11, 0, 1, 2, 99, 0, 0]
    lengths[2] = 100  # a request at the end of its slot
    graph.replay()
    assert start.tolist() == [0, 0, 0, 0] and int(pool[3]) == -1 and slots.tolist() == [-1] * 8


@pytest.mark.parametrize("requests,block", [(1, 16), (5, 8)])
def test_no_parents_at_all(requests, block):
    """An empty list of parents is none for any row, not a chain: rows are refused, and without rows the masks are zero."""
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    tables, held, pool = torch.zeros(requests, 4, dtype=torch.int32, device="cuda"), i32([0] * requests), K.block_pool(9, "cuda")
    none, lengths = i32([]), i32([0] * requests)
    for mine in (none, i32([7])[1:]):
        torch.full((6 * 2,), 0x5a5a5a5a, dtype=torch.int32, device="cuda")  # (what a result without a store may hold)
        start, slots, positions, mask = K.block_tables(tables, held, pool, lengths, i32([1] * requests), block, 6, parents=mine, max_new=40)
        assert int(pool[3]) == -2 and start.tolist() == [0] * (requests + 1) and slots.tolist() == [-1] * 6
        assert positions.tolist() == [0] * 6 and mask.tolist() == [[0, 0]] * 6
        assert held.tolist() == [0] * requests and int(pool[1]) == 9
        torch.full((6 * 2,), 0x5a5a5a5a, dtype=torch.int32, device="cuda")
        start, slots, positions, mask = K.block_tables(tables, held, pool, lengths, i32([0] * requests), block, 6, parents=mine, max_new=40)
        assert int(pool[3]) == 0 and start.tolist() == [0] * (requests + 1) and slots.tolist() == [-1] * 6
        assert positions.tolist() == [0] * 6 and mask.tolist() == [[0, 0]] * 6
        assert K.block_tables(tables, held, pool, lengths, i32([0] * requests), block, 0, parents=mine)[3].shape == (0, 1)


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("max_rows", [0, 5])
def test_tables_of_no_requests(max_rows, tree):
    """A step without requests has no rows; tree_attn and tree_commit take what comes back."""
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    pool = K.block_pool(3, "cuda")
    pool[3] = -2  # (of the call before)
    tables, none = torch.zeros(0, 4, dtype=torch.int32, device="cuda"), i32([])
    parents = i32([0] * max_rows) if tree else None
    start, slots, positions, mask = K.block_tables(tables, i32([]), pool, none, none, 16, max_rows, parents=parents, max_new=40)
    assert start.tolist() == [0] and start.dtype is torch.int32 and slots.tolist() == [-1] * max_rows and slots.dtype is torch.int64
    assert positions.tolist() == [0] * max_rows and positions.dtype is torch.int32
    assert mask is None if not tree else mask.tolist() == [[0, 0]] * max_rows and mask.dtype is torch.int32
    assert pool.tolist() == [0, 3, 0, 0, 0, 1, 2]
    kv = torch.zeros(1, 2, 3, 2, 16, 64, device="cuda").half()
    q = torch.ones(max_rows, 14, 64, device="cuda").half()
    assert torch.equal(K.tree_attn(q, kv[0, 0], kv[0, 1], tables, none, start, mask=mask, out=q), torch.ones_like(q))
    path, accepted, following, after = K.tree_commit(kv, tables, none, start, i32([0] * max_rows), slots, slots, 4)
    assert path.shape == (0, 4) and accepted.shape == following.shape == after.shape == (0,)


# ---- tree_commit -------------------------------------------------------------------------------
def _walk(parents, tokens, targets):
    path, at = [0], 0
    while True:
        nexts = [i for i in range(at + 1, len(parents)) if parents[i] == at and tokens[i] == targets[at]]
        if not nexts:
            return path
        at = nexts[0]
        path.append(at)


@pytest.mark.parametrize("wide", [torch.int32, torch.int64])
@pytest.mark.parametrize("new,block,layers,kv_heads,dim,dtype", [
    ([1], 16, 1, 1, 64, torch.float16), ([5, 0, 9, 1], 16, 3, 2, 64, torch.float16), ([40, 64, 33], 8, 2, 8, 128, torch.bfloat16),
    ([200, 7], 300, 2, 2, 64, torch.float16), ([12] * 20, 4, 24, 2, 64, torch.float16), ([6, 6], 16, 2, 3, 40, torch.bfloat16)])
def test_commit(new, block, layers, kv_heads, dim, dtype, wide):
    g = torch.Generator().manual_seed(sum(new))
    lengths = [int(torch.randint(0, 50, (1,), generator=g)) for _ in new]
    counts = [max(1, -(-(n + m) // block)) for n, m in zip(lengths, new)]
    ids = torch.randperm(sum(counts) + 2, generator=g).tolist()
    tables = [[ids.pop() for _ in range(c)] for c in counts]
    kv = torch.randn(layers, 2, sum(counts) + 2, kv_heads, block, dim, generator=g).to(dtype)
    starts, parents, tokens, targets = [0], [], [], []
    for b, n in enumerate(new):
        tree = [-1] + [int(torch.randint(max(0, i - 3), i, (1,), generator=g)) for i in range(1, n)] if n else []
        parents += tree
        tokens += torch.randint(0, 3, (n,), generator=g).tolist()  # (few tokens: many agree, siblings too)
        targets += torch.randint(0, 3, (n,), generator=g).tolist()
        starts.append(starts[-1] + n)
    want, paths = kv.clone(), []
    for b, n in enumerate(new):
        s = slice(starts[b], starts[b + 1])
        path = _walk(parents[s], tokens[s], targets[s]) if n else []
        paths.append(path)
        for j, node in enumerate(path):
            p, t = lengths[b] + node, lengths[b] + j
            want[:, :, tables[b][t // block], :, t % block] = kv[:, :, tables[b][p // block], :, p % block]
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    width = max(counts)
    dev = kv.cuda()
    got = K.tree_commit(dev, i32([t + [-1] * (width - len(t)) for t in tables]), i32(lengths), i32(starts), i32(parents),
                        torch.tensor(tokens, dtype=wide, device="cuda"), torch.tensor(targets, dtype=wide, device="cuda"), max(new))
    path, accepted, nxt, after = (t.tolist() for t in got)
    assert got[2].dtype is wide
    assert accepted == [len(p) for p in paths] and after == [n + len(p) for n, p in zip(lengths, paths)]
    assert path == [p + [-1] * (max(new) - len(p)) for p in paths]
    assert nxt == [targets[starts[b] + p[-1]] if p else -1 for b, p in enumerate(paths)]
    assert torch.equal(dev.cpu(), want)


def test_commit_moves_a_long_chain():
    """A path of 1000 of 1024 nodes that all move by one or more, each onto the place that the one before it leaves."""
    n, block = 1024, 16
    parents = [-1, 0] + [0] + [i - 1 for i in range(3, n)]  # node 1 is wrong, node 2 the chain's next
    tokens = [0, 9] + list(range(10, n + 8))
    targets = [10, 5] + list(range(11, n + 9))
    targets[1001] = 3
    kv = torch.randn(2, 2, 70, 2, block, 64, device="cuda", generator=_gen(4)).half()
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    tables = torch.randperm(70, generator=torch.Generator().manual_seed(1))[:66].view(1, 66).to("cuda", torch.int32)
    line = kv[:, :, tables[0].long()].transpose(3, 4).flatten(2, 3)  # [2, 2, positions, heads, dim]
    path, accepted, _, _ = K.tree_commit(kv, tables, i32([21]), i32([0, n]), i32(parents), i32(tokens), i32(targets), n)
    assert int(accepted) == 1001 and path[0, :4].tolist() == [0, 2, 3, 4]
    after = kv[:, :, tables[0].long()].transpose(3, 4).flatten(2, 3)
    assert torch.equal(after[:, :, :22], line[:, :, :22])
    assert torch.equal(after[:, :, 22:22 + 1000], line[:, :, 23:23 + 1000])
    assert torch.equal(after[:, :, 22 + 1000:], line[:, :, 22 + 1000:])


def test_commit_leaves_bad_requests_alone():
    kv = torch.randn(1, 2, 4, 2, 16, 64, device="cuda", generator=_gen(5)).half()
    before = kv.clone()
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")
    # a tree larger than max_new; blocks that are not there
    got = K.tree_commit(kv, i32([[0, 1], [-1, 99]]), i32([3, 14]), i32([0, 5, 8]), i32([-1, 0, 1, 2, 3, -1, 0, 0]),
                        i32([1, 1, 1, 1, 1, 1, 2, 1]), i32([1] * 8), 4)
    assert got[1].tolist() == [0, 2] and got[3].tolist() == [3, 16] and got[0].tolist() == [[-1] * 4, [0, 2, -1, -1]]
    assert got[2].tolist() == [-1, 1]
    assert torch.equal(kv, before)


def test_two_threads_of_tables_and_commits():
    """Steps of two threads with a pool and a cache each, on one stream: blocks, rows and masks, then the commit."""
    i32 = functools.partial(torch.tensor, dtype=torch.int32, device="cuda")

    def steps(seed, out, start=None):
        kv = torch.randn(2, 2, 20, 2, 16, 64, device="cuda", generator=_gen(seed)).half()
        tables, held, lengths = torch.zeros(4, 5, dtype=torch.int32, device="cuda"), i32([0] * 4), i32([0] * 4)
        pool, new = K.block_pool(20, "cuda"), i32([3, 1, 0, 6])
        parents, tokens = i32([-1, 0, 0, -1, -1, 0, 0, 1, 2, 2]), i32([0, seed, 1, 0, 0, 1 - seed, seed, 1, 1, 0])
        targets = i32([1] * 10)
        torch.cuda.synchronize()
        if start is not None:
            start.wait()
        for _ in range(60):
            row_start, slots, positions, mask = K.block_tables(tables, held, pool, lengths, new, 16, 10, parents=parents, max_new=6)
            more = K.tree_commit(kv, tables, lengths, row_start, parents, tokens, targets, 6)
            out.append([row_start, slots, positions, mask, *more])
            lengths = more[3] % 60
        out.append([tables, held, pool, lengths, kv])

    want, got = [[], []], [[], []]
    for seed in range(2):
        steps(seed, want[seed])
    start = threading.Barrier(2)
    threads = [threading.Thread(target=steps, args=(seed, got[seed], start)) for seed in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert len(a) == len(b) == 61
        for x, y in zip(a, b):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


# ---- together ------------------------------------------------------------------------------------
def test_a_run_of_them_together():
    """Five steps of drafted trees over a pool: blocks, places and masks, the append, attention, the commit.  The rows of K and V
    carry their token and position, so the cache can be read back: after every step it holds each request's text in order, and
    attention is that of the text and the node's branch."""
    heads, kv_heads, dim, block, layers, requests, width = 14, 2, 64, 8, 2, 6, 16
    table = torch.randn(2, 50, kv_heads, dim, device="cuda", generator=_gen(1)).half()  # K and V of a token
    kv = torch.full((layers, 2, 60, kv_heads, block, dim), float("nan"), device="cuda", dtype=torch.float16)
    tables = torch.zeros(requests, width, dtype=torch.int32, device="cuda")
    held, lengths = (torch.zeros(requests, dtype=torch.int32, device="cuda") for _ in range(2))
    pool = K.block_pool(60, "cuda")
    texts, g = [[] for _ in range(requests)], torch.Generator().manual_seed(3)
    for step in range(5):
        new = [0 if (b + step) % 5 == 4 else 1 + (7 * b + 3 * step) % 11 for b in range(requests)]
        trees = [_random_parents(n, 10 * step + b) if n else [] for b, n in enumerate(new)]
        rows = sum(new)
        parents = torch.tensor([p for t in trees for p in t] + [0] * 3, dtype=torch.int32, device="cuda")
        n_new = torch.tensor(new, dtype=torch.int32, device="cuda")
        start, slots, positions, mask = K.block_tables(tables, held, pool, lengths, n_new, block, rows + 3, parents=parents, max_new=11)
        assert int(pool[3]) == 0
        tokens = torch.randint(0, 50, (rows,), generator=g)
        targets = torch.randint(0, 50, (rows,), generator=g)
        first = [sum(new[:b]) for b in range(requests)]
        for b, t in enumerate(trees):  # the target agrees with some child of most nodes
            for i in range(1, new[b]):
                if (i + step) % 4:
                    targets[first[b] + t[i]] = tokens[first[b] + i]
        tokens, targets = tokens.cuda(), targets.cuda()
        flat = kv.permute(2, 4, 0, 1, 3, 5)  # [blocks, block, layers, 2, heads, dim]
        at = slots[:rows]
        flat[at // block, at % block] = table[:, tokens].transpose(0, 1)[:, None].expand(-1, layers, -1, -1, -1)
        q = torch.randn(rows + 3, heads, dim, device="cuda", generator=_gen(step)).half()
        for layer in range(layers):
            got = K.tree_attn(q, kv[layer, 0], kv[layer, 1], tables, lengths, start, mask=mask, max_new=11)
            for b, t in enumerate(trees):
                for i in range(new[b]):
                    branch = [int(tokens[first[b] + j]) for j in sorted(_ancestors(t, i))]
                    assert int(positions[first[b] + i]) == len(texts[b]) + len(branch) - 1
                    k, v = table[:, texts[b] + branch].double().transpose(1, 2)
                    p = torch.softmax(q[first[b] + i].double().view(2, 7, dim) @ k.transpose(1, 2) / 8, -1)
                    assert (got[first[b] + i].double().view(2, 7, dim) - p @ v).abs().max() < 6e-3
        path, accepted, nxt, after = K.tree_commit(kv, tables, lengths, start, parents[:rows], tokens, targets, 11)
        for b, t in enumerate(trees):
            if not new[b]:
                assert int(accepted[b]) == 0
                continue
            s = slice(first[b], first[b] + new[b])
            want = _walk(t, tokens[s].tolist(), targets[s].tolist())
            assert path[b, :len(want)].tolist() == want and int(nxt[b]) == int(targets[first[b] + want[-1]])
            texts[b] += [int(tokens[first[b] + j]) for j in want]
        lengths.copy_(after)
        assert lengths.tolist() == [len(t) for t in texts]
        for b, text in enumerate(texts):
            for p, token in enumerate(text):
                assert torch.equal(kv[:, :, int(tables[b, p // block]), :, p % block], table[:, token].expand(layers, -1, -1, -1))
    over = torch.full((requests,), -1, dtype=torch.int32, device="cuda")
    K.block_tables(tables, held, pool, lengths, over, block, 0)
    assert int(pool[1]) == 60 and held.tolist() == [0] * requests


# ---- the append ----------------------------------------------------------------------------------
def test_append_at_places_apart_from_positions():
    rows, blocks, block = 9, 7, 5
    qkv = torch.randn(rows, 1152, device="cuda", generator=_gen(1)).half()
    cos, sin = K.rope().init_table(torch.rand(32, device="cuda", generator=_gen(2)), 64)
    positions = torch.tensor([3, 4, 4, 5, 0, 63, 64, 70, 2], dtype=torch.int32, device="cuda")
    places = [12, 13, 30, 0, 34, 5, -1, 35, 20]
    kc, vc = (torch.full((blocks, 2, block, 64), 3.0, device="cuda", dtype=torch.float16) for _ in range(2))
    q = K.qkv_rope_append_at(qkv, torch.tensor(places, device="cuda"), positions, cos, sin, kc, vc)
    k2, v2 = (torch.zeros(rows, 2, 80, 64, device="cuda", dtype=torch.float16) for _ in range(2))
    want = K.qkv_rope_append(qkv, torch.arange(rows, dtype=torch.int32, device="cuda"), positions, cos, sin, k2, v2)
    assert torch.equal(q, want)
    keep_k, keep_v = torch.full_like(kc, 3.0), torch.full_like(vc, 3.0)
    for r, p in enumerate(places):
        if 0 <= p < blocks * block:
            keep_k[p // block, :, p % block] = k2[r, :, int(positions[r])]
            keep_v[p // block, :, p % block] = v2[r, :, int(positions[r])]
    assert torch.equal(kc, keep_k) and torch.equal(vc, keep_v)
