"""Sequences that share a prompt, on the GPU, against plain fp64 implementations (ops/reference.py).

Attention outputs are bounded element by element.  P is rounded to bf16 before it meets V and the result once at the
end, each by at most 2^-8 relative, so |out - exact| <= 2^-8 (sum_j p_j |v_j| / l + |exact|); fp32 accumulation of
scores and sums adds below 2^-12 of the first term (128 products, then up to 2^14 keys, 2^-24 each, averaged).
Tokens, tables, counts and copied pages have to be equal.
"""
import pytest
import torch

from bloom_b200 import ops
from bloom_b200.ops import reference as ref

pytestmark = pytest.mark.gpu
BAD = 8  # kStatusBadArgument


@pytest.fixture(autouse=True)
def _status_clean():
    ops.status().zero_()
    yield
    torch.cuda.synchronize()
    assert int(ops.status()[0].item()) == 0, "kernel reported an error"


def took_bits():
    v = int(ops.status()[0].item())
    ops.status().zero_()
    return v


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- attention
class Batch:
    """Groups over a paged cache; every slot behind a sequence's end, and every unused page, holds NaN."""

    def __init__(self, heads, sizes, prefix, own, q_len=1, seed=0, extra_width=0, layers=1, layer=0):
        self.nq, self.nkv, self.D = heads
        g = torch.Generator().manual_seed(seed)
        self.q_len, self.layer = q_len, layer
        self.sizes, self.prefix = list(sizes), list(prefix)
        B = sum(sizes)
        lens = [p + own[(i + sum(sizes[:gi])) % len(own)] for gi, (n, p) in enumerate(zip(sizes, prefix)) for i in range(n)]
        self.width = max((n + 15) // 16 for n in lens) + extra_width
        blocks = sum((n + 15) // 16 for n in lens) + 5
        free = torch.randperm(blocks, generator=g).tolist()
        cache = torch.full((layers, blocks, 2, self.nkv, 16, self.D), float("nan"))
        table, b = [], 0
        for n, p in zip(self.sizes, self.prefix):
            common = [free.pop() for _ in range(p // 16)]
            shared_kv = torch.randn(2, self.nkv, p, self.D, generator=g)
            for _ in range(n):
                row = common + [free.pop() for _ in range((lens[b] + 15) // 16 - p // 16)]
                kv = torch.cat([shared_kv, torch.randn(2, self.nkv, lens[b] - p, self.D, generator=g)], 2)
                for j, page in enumerate(row):
                    part = kv[:, :, 16 * j:16 * (j + 1)]
                    cache[layer, page, :, :, :part.shape[2]] = part
                table.append(row + [0] * (self.width - len(row)))
                b += 1
        self.cache = cache.bfloat16().cuda()
        self.table, self.lens = i32(table), i32(lens)
        self.q = torch.randn(B * q_len, self.nq, self.D, generator=g).bfloat16().cuda()
        self.scale = self.D ** -0.5
        self.plan = ops.shared_prefix_plan(self.sizes, self.prefix, num_q_heads=self.nq, num_kv_heads=self.nkv,
                                           head_dim=self.D, q_len=q_len, max_seq_len=max(lens), device="cuda")

    def run(self, out=None, lens=None):
        out = torch.full_like(self.q, 7.0) if out is None else out
        return ops.shared_prefix_attention(self.q, self.cache, self.layer, self.table,
                                           self.lens if lens is None else lens, out, plan=self.plan, scale=self.scale)

    def check(self, out, lens=None, q=None):
        lens = self.lens if lens is None else lens
        want, mag = ref.paged_attention(self.q if q is None else q, self.cache[self.layer], self.table, lens,
                                        self.q_len, self.scale)
        bound = 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -12 * mag
        err = (out.double() - want).abs()
        assert bool((err <= bound).all()), f"off by {float((err - bound).max()):.3g}, {int((err > bound).sum())} values"


HEADS = [(32, 8, 128), (8, 8, 64), (9, 3, 64), (16, 1, 128), (4, 2, 128), (64, 8, 128), (33, 1, 64), (71, 1, 128)]


@pytest.mark.parametrize("heads", HEADS)
@pytest.mark.parametrize("sizes,prefix,own", [
    ([1], [1], [1]), ([1], [16], [1]), ([2], [15], [2, 17]), ([4], [128], [1, 16, 33]), ([3, 1, 5], [100, 0, 257], [1, 40]),
    ([40], [300], [3, 16, 64, 1]), ([1, 1], [0, 0], [1, 200]), ([70, 2], [129, 1000], [5, 1])])
def test_shared_prefix_attention(heads, sizes, prefix, own):
    b = Batch(heads, sizes, prefix, own, seed=len(sizes))
    b.check(b.run())


@pytest.mark.parametrize("q_len", [2, 3, 4, 8])
@pytest.mark.parametrize("heads", [(32, 8, 128), (9, 3, 64), (8, 1, 128)])
def test_verify_rows(q_len, heads):
    b = Batch(heads, [5, 1, 17], [130, 64, 33], [q_len, q_len + 1, 50], q_len=q_len, seed=q_len)
    b.check(b.run())


@pytest.mark.parametrize("heads,sizes,prefix,own", [((8, 2, 128), [2], [4100], [1, 3000]), ((8, 2, 64), [3], [0], [5000]),
                                                    ((32, 8, 128), [130], [2500], [1, 30]),
                                                    ((4, 4, 128), [1, 300], [9000, 64], [600, 2])])
def test_long(heads, sizes, prefix, own):
    b = Batch(heads, sizes, prefix, own, seed=3)
    b.check(b.run())


@pytest.mark.parametrize("q_len", [1, 4])
def test_no_member_of_its_own_tokens(q_len):
    """seq_len == prefix: nothing but the prefix; verify rows then see less than all of it."""
    b = Batch((8, 2, 128), [6], [200], [0], q_len=q_len)
    b.check(b.run())


def test_ended_and_short_members():
    b = Batch((8, 2, 128), [5, 4, 3], [96, 48, 64], [20, 1, 33])
    ended = b.lens.clone()
    ended[0] = 0  # the member whose row the prefix would be read through first
    ended[5:9] = 0  # a whole group
    ended[10] = 40  # shorter than its prefix: sees what it holds of it
    b.table[0] = 0
    ended_out = b.run(lens=ended)
    b.check(ended_out, lens=ended)
    assert bool((ended_out[0] == 0).all()) and bool((ended_out[5:9] == 0).all())
    b.check(b.run(lens=torch.zeros_like(ended)), lens=torch.zeros_like(ended))


def test_strides_and_layer():
    b = Batch((8, 2, 64), [4, 9], [50, 130], [7, 16], layers=3, layer=2, extra_width=5)
    wide = torch.zeros(13, 20, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, 3:11] = b.q
    out = torch.full((13, 24, 64), 3.0, device="cuda", dtype=torch.bfloat16)
    table = torch.full((13, b.table.shape[1] + 3), -9, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table
    ops.shared_prefix_attention(wide[:, 3:11], b.cache, 2, table[:, :b.table.shape[1]], b.lens, out[:, 8:16],
                                plan=b.plan, scale=b.scale)
    b.check(out[:, 8:16])
    assert bool((out[:, :8] == 3).all()) and bool((out[:, 16:] == 3).all())


@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 8.0])
@pytest.mark.parametrize("members", [5, 20, 40])
def test_scales(scale, members):
    b = Batch((8, 2, 128), [members], [150], [1, 30])
    b.scale = scale
    b.check(b.run())


def test_matches_plain_decode_of_the_same_tables():
    b = Batch((32, 8, 128), [16], [512], [1, 40, 100])
    b.cache = torch.nan_to_num(b.cache)
    plain = torch.empty_like(b.q)
    ops.paged_decode_attention(b.q, b.cache, 0, b.table, b.lens, plain, scale=b.scale)
    # each is within its own roundings of the same exact values
    want, mag = ref.paged_attention(b.q, b.cache[0], b.table, b.lens, 1, b.scale)
    bound = 2 * (2.0 ** -8 * (mag + want.abs()) + 2.0 ** -12 * mag)
    assert bool(((b.run().double() - plain.double()).abs() <= bound).all())


def test_no_sequences():
    plan = ops.shared_prefix_plan([], [], num_q_heads=8, num_kv_heads=2, head_dim=64, device="cuda")
    q = torch.zeros(0, 8, 64, device="cuda", dtype=torch.bfloat16)
    cache = torch.zeros(1, 2, 2, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    out = ops.shared_prefix_attention(q, cache, 0, i32([]).view(0, 3), i32([]), torch.empty_like(q), plan=plan, scale=1.0)
    assert out.shape == q.shape


def test_bad_ids_set_the_status():
    """The cache handed over is the front half of a larger one, and ids outside it are not followed."""
    b = Batch((8, 2, 128), [3], [64], [20])
    b.cache = torch.nan_to_num(b.cache)
    b.table[1, 5] = b.cache.shape[1] + 3
    b.run()
    assert took_bits() == BAD
    b.table[1, 5] = -1
    b.run()
    assert took_bits() == BAD
    b.table[1, 5] = 0
    b.run(lens=b.lens + 16 * b.width)
    assert took_bits() == BAD
    b.run(lens=b.lens - 1000)
    assert took_bits() == BAD


def test_graph_replay_and_two_streams():
    b, c = Batch((32, 8, 128), [20, 3], [300, 77], [1, 20], seed=1), Batch((9, 3, 64), [40], [200], [9, 2], seed=2)
    outs = [torch.empty_like(b.q), torch.empty_like(b.q), torch.empty_like(c.q)]
    b.run(outs[0]), c.run(outs[2])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.run(outs[1])
        c.run(outs[2])
    b.q.copy_(torch.randn_like(b.q))
    c.q.copy_(torch.randn_like(c.q))
    b.lens -= 1
    for _ in range(3):
        for o in outs:
            o.fill_(9)
        g.replay()
        b.check(outs[1])
        c.check(outs[2])
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(10):
        with torch.cuda.stream(s):
            b.run(outs[0])
        with torch.cuda.stream(t):
            b.run(outs[1])
            c.run(outs[2])
    torch.cuda.synchronize()
    b.check(outs[0])
    assert torch.equal(outs[0], outs[1])
    c.check(outs[2])


def test_large_groups_in_graphs_and_on_many_streams():
    """Prefix and suffixes run on two streams there: calls from 40 streams of the pool, captured and eager."""
    b = Batch((32, 8, 128), [70, 2], [400, 130], [1, 20, 90], seed=4)
    want = b.run()
    b.check(want)
    outs = [torch.empty_like(b.q) for _ in range(40)]
    torch.cuda.synchronize()
    for out in outs:
        with torch.cuda.stream(torch.cuda.Stream()):
            b.run(out)
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)
    graphs = []
    for out in outs[:2]:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            b.run(out)
            b.run(out)
    outs[0].fill_(3), outs[1].fill_(3)
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s):
            graphs[0].replay()
        with torch.cuda.stream(t):
            graphs[1].replay()
        b.run(outs[2])
    torch.cuda.synchronize()
    for out in outs[:3]:
        assert torch.equal(out, want)


@pytest.mark.parametrize("members", [3, 9, 20, 70])
def test_queries_before_the_first_token(members):
    """Verify rows of sequences shorter than q_len: positions before the first token see nothing and give zeros."""
    b = Batch((32, 8, 128), [members], [40], [4, 30], q_len=4)
    lens = b.lens.clone()
    lens[::2] = 2
    out = b.run(lens=lens)
    b.check(out, lens=lens)
    assert bool((out.view(members, 4, 32, 128)[::2, :2] == 0).all())


# ---------------------------------------------------------------- pages
def page_state(kind, lens, seed=0, spare=6, layers=2):
    g = torch.Generator().manual_seed(seed)
    width = max((n + 15) // 16 for n in lens) + 2
    blocks = sum((n + 15) // 16 for n in lens) + spare
    shape = {"bf16": (2, 3, 16, 64), "int8": (2 * 2 * 16 * 132,), "wide": (2 * 2 * 16 * 256 + 8,),
             "tiny": (16,)}[kind]
    dt = {"bf16": torch.bfloat16, "int8": torch.uint8, "wide": torch.bfloat16, "tiny": torch.uint8}[kind]
    cache = (torch.randn(layers, blocks, *shape, generator=g).bfloat16() if dt == torch.bfloat16
             else torch.randint(0, 256, (layers, blocks, *shape), generator=g, dtype=dt)).cuda()
    free = torch.randperm(blocks, generator=g).tolist()
    table, count = [], [0] * blocks
    for n in lens:
        row = [free.pop() for _ in range((n + 15) // 16)]
        for p in row:
            count[p] += 1
        table.append(row + [0] * (width - len(row)))
    return cache, i32(table), i32(lens), i32(count), free


def check_fork(args):
    want = [t.clone() for t in args]
    table, lens = ref.kv_fork(*want)
    got = ops.kv_fork(*args)
    assert torch.equal(got[0], table) and torch.equal(got[1], lens)
    for a, w in zip(args, want):  # the cache and the counts as they should be, the rest untouched
        assert torch.equal(a, w)
    return got


@pytest.mark.parametrize("kind", ["bf16", "int8", "wide", "tiny"])
@pytest.mark.parametrize("lens,parents", [([1], [0]), ([16], [0, 0]), ([17, 0, 33], [0, 1, 2, 2, 2]), ([15, 32], [-1, 1, 0]),
                                          ([250, 31, 64, 5], [3, 3, 2, 0, 0, 0, 1, -7])])
def test_kv_fork(kind, lens, parents):
    cache, table, n, count, free = page_state(kind, lens, spare=len(parents) + 3)
    check_fork((cache, table, n, i32(parents), i32(free[:len(parents)]), count))


def test_kv_fork_of_a_fork_and_none():
    cache, table, n, count, free = page_state("bf16", [40, 7])
    t2, n2 = check_fork((cache, table, n, i32([0, 1]), i32(free[:2]), count))
    check_fork((cache, t2, n2, i32([1, 0, 0]), i32(free[2:5]), count))
    t, m = ops.kv_fork(cache, table, n, i32([]), i32([]), count)
    assert t.shape == (0, table.shape[1]) and m.shape == (0,)


def test_kv_fork_takes_no_fresh_page_where_the_last_is_full():
    cache, table, n, count, _ = page_state("bf16", [32])
    check_fork((cache, table, n, i32([0, 0]), i32([-1, 10**9]), count))


@pytest.mark.parametrize("kw", ["parent", "fresh", "taken", "twice", "page", "length"])
def test_kv_fork_bad_ids_set_the_status(kw):
    cache, table, n, count, free = page_state("bf16", [20, 40])
    parents, fresh = i32([0, 1]), i32(free[:2])
    if kw == "parent":
        parents[1] = 2
    elif kw == "fresh":
        fresh[1] = cache.shape[1]
    elif kw == "taken":
        fresh[1] = table[0, 0]
    elif kw == "twice":
        fresh[1] = fresh[0]
    elif kw == "page":
        table[1, 1] = -4
    else:
        n[1] = 16 * table.shape[1] + 1
    ops.kv_fork(cache, table, n, parents, fresh, count)
    assert took_bits() == BAD


def test_kv_free():
    cache, table, n, count, free = page_state("bf16", [20, 0, 33, 16, 1])
    t2, n2 = ops.kv_fork(cache, table, n, i32([2, 2]), i32(free[:2]), count)
    table, n = torch.cat([table, t2]), torch.cat([n, n2])
    for rows in ([2, -1, 1], [2, 2, 5, 5, 0], [], list(range(7))):
        w = [t.clone() for t in (table, n, count)]
        ref.kv_free(w[0], w[1], torch.tensor(rows), w[2])
        ops.kv_free(table, n, i32(rows), count)
        assert torch.equal(table, w[0]) and torch.equal(n, w[1]) and torch.equal(count, w[2])
    assert int(count.abs().sum()) == 0


def test_kv_free_bad_ids_set_the_status():
    _, table, n, count, _ = page_state("bf16", [20, 40])
    ops.kv_free(table, n, i32([2]), count)
    assert took_bits() == BAD
    table[0, 0] = 10**6
    ops.kv_free(table, n, i32([0]), count)
    assert took_bits() == BAD
    count.zero_()
    ops.kv_free(table, n, i32([1]), count)
    assert took_bits() == BAD and int(count.abs().sum()) == 0


@pytest.mark.parametrize("kind", ["bf16", "int8", "wide", "tiny"])
@pytest.mark.parametrize("lens,done,spare", [([1], [], 0), ([1], [0], 0), ([40, 17, 300, 1], [0, 2], 3), ([200] * 9, [1, 3, 4], 70),
                                             ([16] * 64, [], 0), ([5] * 33, list(range(0, 33, 2)), 31)])
def test_kv_compact(kind, lens, done, spare):
    cache, table, n, count, free = page_state(kind, lens, spare=spare, seed=spare)
    if spare:  # two rows share pages
        t2, n2 = ops.kv_fork(cache, table, n, i32([len(lens) - 1]), i32(free[:1]), count)
        table, n = torch.cat([table, t2]), torch.cat([n, n2])
    ops.kv_free(table, n, i32(done), count)
    args = (cache, table, n, count)
    want = [t.clone() for t in args]
    moved, used = ref.kv_compact(*want)
    got = ops.kv_compact(*args)
    assert torch.equal(got[0], moved) and torch.equal(got[1], used)
    for a, w in zip(args, want):
        assert torch.equal(a, w)


@pytest.mark.parametrize("blocks", [1, 31, 33, 8191, 50000, 400001])
def test_kv_compact_many_pages(blocks):
    g = torch.Generator(device="cuda").manual_seed(blocks)
    cache = torch.randint(0, 2**31 - 1, (1, blocks, 4), generator=g, device="cuda", dtype=torch.int32)
    count = (torch.rand(blocks, generator=g, device="cuda") < 0.4).int() * 3
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    old, old_count = cache.clone(), count.clone()
    moved, used = ops.kv_compact(cache, table, i32([0]), count)
    held = (old_count > 0).nonzero()[:, 0]
    assert int(used) == held.numel() and bool((moved[old_count <= 0] == -1).all())
    assert torch.equal(moved[held].sort()[0], torch.arange(int(used), device="cuda", dtype=torch.int32))
    assert torch.equal(cache[:, moved[held].long()], old[:, held])
    low = held[held < int(used)]
    assert torch.equal(moved[low].long(), low)
    high = moved[held[held >= int(used)]]
    assert bool((high[1:] > high[:-1]).all())  # both in rising order
    assert torch.equal(count, (torch.arange(blocks, device="cuda") < used).int() * 3)


def test_kv_compact_bad_ids_set_the_status():
    cache, table, n, count, _ = page_state("bf16", [40, 20])
    table[0, 1] = -1
    ops.kv_compact(cache, table, n, count)
    assert took_bits() == BAD
    cache, table, n, count, free = page_state("bf16", [40, 20])
    table[0, 1] = free[0]  # a page that nothing holds
    ops.kv_compact(cache, table, n, count)
    assert took_bits() == BAD


# ---------------------------------------------------------------- draws
def check_draw(logits, u, temperature, **kw):
    def f(v, dt=torch.float32):
        return torch.tensor(v, dtype=dt, device="cuda")

    B = logits.shape[0]
    t = f(temperature * B if len(temperature) == 1 else temperature)
    kw = {k: f(v * B if len(v) == 1 else v, torch.int32 if k == "top_k" else torch.float32) for k, v in kw.items()}
    got = ops.sample_uniform(logits, u, t, **kw)
    want = ref.sample_uniform(logits, u, t, **kw)
    assert torch.equal(got.cpu(), want), (got.cpu() != want).nonzero()[:5].tolist()
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [1, 2, 7, 255, 256, 257, 1000, 4097, 8192, 32001, 49152, 128257, 151936, 262144])
def test_sample_uniform(V, dtype):
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = (torch.randn(9, V, generator=g, device="cuda") * 3).to(dtype)
    u = torch.rand(9, 3, generator=g, device="cuda")
    check_draw(logits, u, [0.7])
    check_draw(logits, u, [1.0], top_k=[0, 1, 2, 3, 50, V, V + 1, 1000, -1])
    check_draw(logits, u, [1.0], top_p=[0.1, 0.5, 0.9, 0.95, 0.999, 1.0, 0.0, 1.5, 0.3])
    check_draw(logits, u, [1.3], min_p=[0.0, 0.01, 0.1, 0.5, 1.0, 2.0, -1.0, 0.05, 0.9])
    check_draw(logits, u, [0.0, 0.2, 1.0, 2.0, -1.0, 0.05, 5.0, 0.6, 0.9], top_k=[40], top_p=[0.9], min_p=[0.02])
    check_draw(logits, u[:, 0].contiguous(), [0.8], top_p=[0.9])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3, 600, 5000, 70000])
def test_sample_uniform_ties(V, dtype):
    """Few distinct values (all weights well above 2^-46): the cut of top-k / top-p falls inside a tie."""
    g = torch.Generator(device="cuda").manual_seed(V)
    logits = torch.randint(0, 6, (8, V), generator=g, device="cuda").to(dtype)
    logits[1] = 2.0
    logits[2] = -0.0
    logits[2, ::2] = 0.0
    u = torch.rand(8, 40, generator=g, device="cuda")
    u[:, 0] = 0.0
    u[:, 1] = 1.0 - 2.0**-24
    for k in (1, 2, V // 7 + 1, V // 2, V - 1):
        check_draw(logits, u, [1.0], top_k=[k])
    for p in (1e-6, 0.2, 0.5, 0.77, 0.9999):
        check_draw(logits, u, [1.1], top_p=[p])
        check_draw(logits, u, [1.1], top_p=[p], top_k=[V // 3 + 1])
    check_draw(logits, u, [1.0], min_p=[0.2])


def test_sample_uniform_masks_and_specials():
    inf = float("inf")
    g = torch.Generator(device="cuda").manual_seed(5)
    logits = torch.randn(10, 3001, generator=g, device="cuda")
    logits[0] = -inf
    logits[1] = float("nan")
    logits[2, :-1] = -inf
    logits[3, 5::7] = float("nan")
    logits[4, 100] = logits[4, 2000] = inf
    logits[5] = torch.finfo(torch.float32).min
    logits[6, 17:] = torch.finfo(torch.float32).min
    logits[7] *= 1e-30
    logits[8] *= 1e5
    logits[9, :2900] = -inf
    u = torch.rand(10, 6, generator=g, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        x = logits.to(dtype)
        for t in (1.0, 0.0, 1e-3, 1e4):
            got = check_draw(x, u, [t])
            assert bool((got[:2] == -1).all()) and bool((got[2] == 3000).all())
            check_draw(x, u, [t], top_k=[50])
            check_draw(x, u, [t], top_k=[2950], top_p=[0.9])
            check_draw(x, u, [t], top_p=[0.8], min_p=[0.1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_uniform_strides_and_one_row(dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    wide = (torch.randn(12, 20011, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(12, 9, generator=g, device="cuda")
    check_draw(wide[:, 1:20000], u[:, 2:7], [0.9], top_p=[0.9], top_k=[100])
    check_draw(wide[::3, 3:], u[::3], [0.9], top_k=[7])
    check_draw(wide[5:6], u[5:6], [1.0], top_p=[0.6])
    check_draw(wide[:0], u[:0], [1.0])
    assert ops.sample_uniform(wide, u[:, :0], torch.ones(12, device="cuda")).shape == (12, 0)


def test_sample_uniform_follows_the_distribution():
    """Evenly spaced u over the top-p support gives each token its share of the draws, to one draw."""
    logits = torch.log(torch.tensor([[8.0, 4.0, 2.0, 1.0, 1.0]], device="cuda"))
    u = (torch.arange(1400, device="cuda").view(1, -1) + 0.5) / 1400
    got = ops.sample_uniform(logits, u, torch.ones(1, device="cuda"), top_k=i32([3]))
    assert torch.bincount(got[0], minlength=5).tolist() == [800, 400, 200, 0, 0]


def test_sample_uniform_graph_and_repeat():
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.randn(64, 50000, generator=g, device="cuda").bfloat16()
    u, t = torch.rand(64, 2, generator=g, device="cuda"), torch.full((64,), 0.8, device="cuda")
    p = torch.full((64,), 0.9, device="cuda")
    out = torch.empty(64, 2, dtype=torch.int32, device="cuda")
    ops.sample_uniform(logits, u, t, top_p=p, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.sample_uniform(logits, u, t, top_p=p, out=out)
    logits.copy_(torch.randn(64, 50000, generator=g, device="cuda"))
    u.uniform_(generator=g)
    want = ref.sample_uniform(logits, u, t, top_p=p)
    for _ in range(5):
        out.fill_(-5)
        graph.replay()
        assert torch.equal(out.cpu(), want)


# ---------------------------------------------------------------- a run of them together
def test_many_completions_of_one_prompt():
    """Prefill two prompts, fork them, draw each child's first token, decode a few steps with the shared prefix, end
    half of the children, compact, decode on: every step's attention matches a plain fp64 pass over the tables."""
    nq, nkv, D, prompts, per = 8, 2, 128, [70, 33], 5
    g = torch.Generator(device="cuda").manual_seed(0)
    NB, W, vocab = 64, 8, 500
    cache = torch.zeros(1, NB, 2, nkv, 16, D, device="cuda", dtype=torch.bfloat16)
    count = torch.zeros(NB, dtype=torch.int32, device="cuda")
    free = torch.randperm(NB, generator=torch.Generator().manual_seed(1)).tolist()
    cs = ops.rope_cos_sin(256, D, 10000.0, device="cuda")
    rows = []
    for n in prompts:
        pages = [free.pop() for _ in range((n + 15) // 16)]
        count[i32(pages).long()] = 1
        rows.append(pages + [0] * (W - len(pages)))
        qkv = torch.randn(n, (nq + 2 * nkv) * D, generator=g, device="cuda").bfloat16()
        slots = i32([pages[t // 16] * 16 + t % 16 for t in range(n)])
        ops.rope_kv_write(qkv, torch.arange(n, device="cuda"), slots, cs, torch.empty(n, nq, D, device="cuda", dtype=torch.bfloat16),
                          cache, 0, nq, nkv)
    parents = [p for p in range(2) for _ in range(per)]
    table, lens = ops.kv_fork(cache, i32(rows), i32(prompts), i32(parents), i32([free.pop() for _ in parents]), count)
    ops.kv_free(i32(rows), i32(prompts), i32([0, 1]), count)  # the prompts' own rows are not needed any more
    logits = torch.randn(2, vocab, generator=g, device="cuda")
    first = ops.sample_uniform(logits, torch.rand(2, per, generator=g, device="cuda"), torch.ones(2, device="cuda"),
                               min_p=torch.full((2,), 0.05, device="cuda"))
    assert bool(((first >= 0) & (first < vocab)).all())
    plan = ops.shared_prefix_plan([per, per], [n // 16 * 16 for n in prompts], num_q_heads=nq, num_kv_heads=nkv,
                                  head_dim=D, device="cuda")

    def step():
        B = lens.shape[0]
        host = lens.tolist()
        for b, n in enumerate(host):
            if n and n % 16 == 0:  # a new page
                page = free.pop()
                table[b, n // 16] = page
                count[page] = 1
        live = lens > 0
        at = lens.long().clamp(max=16 * W - 1)
        slots = torch.where(live, table.gather(1, (at // 16)[:, None])[:, 0] * 16 + (at % 16).int(), -1).int()
        qkv = torch.randn(B, (nq + 2 * nkv) * D, generator=g, device="cuda").bfloat16()
        q = torch.empty(B, nq, D, device="cuda", dtype=torch.bfloat16)
        ops.rope_kv_write(qkv, at, slots, cs, q, cache, 0, nq, nkv)
        lens.add_(live.int())
        out = ops.shared_prefix_attention(q, cache, 0, table, lens, torch.empty_like(q), plan=plan, scale=D ** -0.5)
        want, mag = ref.paged_attention(q, cache[0], table, lens, 1, D ** -0.5)
        assert bool(((out.double() - want).abs() <= 2.0 ** -8 * (mag + want.abs()) + 2.0 ** -12 * mag).all())
        assert bool((out[~live] == 0).all())

    for _ in range(18):
        step()
    ops.kv_free(table, lens, i32([0, 3, 5, 6, 7]), count)
    moved, used = ops.kv_compact(cache, table, lens, count)
    assert int(used) == int((count > 0).sum()) and bool((count[:int(used)] > 0).all())
    free = list(range(int(used), NB))
    for _ in range(3):
        step()
    ops.kv_free(table, lens, i32(list(range(10))), count)
    assert int(count.abs().sum()) == 0 and int(lens.sum()) == 0


# ---------------------------------------------------------------- the side stream of large groups
def large_batch(seed=6):
    """A group of more than 128 query rows per KV head: prefix and suffixes run side by side on two streams."""
    b = Batch((32, 8, 128), [70, 2], [400, 130], [1, 20, 90], seed=seed)
    assert b.plan.tile_rows == 256
    return b


def test_every_large_group_call_of_a_capture_runs_side_by_side(tmp_path):
    """In a graph of 40 calls (a model's layers) of three kernels each, the longest chain is two kernels a call: prefix
    and suffixes do not wait for one another."""
    import re

    b = large_batch()
    out = torch.empty_like(b.q)
    b.run(out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(g):
        for _ in range(40):
            b.run(out)
    path = tmp_path / "graph.dot"
    g.debug_dump(str(path))
    edges = set(re.findall(r'"([^"]+)"\s*->\s*"([^"]+)"', path.read_text()))
    follow, waits = {}, {}
    for a, z in edges:
        follow.setdefault(a, []).append(z)
        waits[z] = waits.get(z, 0) + 1
    nodes = {n for e in edges for n in e}
    depth = dict.fromkeys(nodes, 1)
    ready = [n for n in nodes if n not in waits]
    while ready:
        n = ready.pop()
        for z in follow.get(n, []):
            depth[z] = max(depth[z], depth[n] + 1)
            waits[z] -= 1
            if waits[z] == 0:
                ready.append(z)
    assert len(nodes) == 120 and max(depth.values()) == 80


def test_capture_of_large_groups_takes_no_stream_of_others():
    """While a capture holds 40 large-group calls, work of another thread on any of PyTorch's streams runs at once and
    is not recorded, an eager call of another thread included."""
    import threading

    b = large_batch()
    want = b.run()
    out, other = torch.empty_like(b.q), torch.full_like(b.q, 5.0)
    streams = [torch.cuda.Stream() for _ in range(32)]
    x = torch.zeros(32, device="cuda")
    x[0].add_(0)
    torch.cuda.synchronize()
    failed, skipped = [], []

    def work(capturing):
        try:
            for i, s in enumerate(streams):
                if s.cuda_stream == capturing:
                    skipped.append(i)
                    continue
                with torch.cuda.stream(s):
                    x[i].add_(1)
                    if i == 3 or (i == 4 and 3 in skipped):
                        b.run(other)
        except Exception as e:  # noqa: BLE001  (shown by the assertion below)
            failed.append(e)

    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, capture_error_mode="thread_local"):
        for _ in range(40):
            b.run(out)
        t = threading.Thread(target=work, args=(torch.cuda.current_stream().cuda_stream,))
        t.start()
        t.join()
        b.run(out)
    torch.cuda.synchronize()
    assert not failed, failed
    ones = torch.ones(32, device="cuda")
    ones[skipped] = 0
    assert torch.equal(x, ones) and torch.equal(other, want)
    out.fill_(3)
    other.fill_(4)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(x, ones) and bool((other == 4).all())


# ---------------------------------------------------------------- children that are refused
@pytest.mark.parametrize("kw", ["parent", "fresh", "taken", "taken by many", "source", "twice", "page", "last page",
                                "length"])
def test_kv_fork_refuses_a_child_and_leaves_the_rest(kw):
    """A child that cannot be made gets an empty row, and nothing is copied, counted or changed for it; the other children
    are made."""
    cache, table, n, count, free = page_state("int8", [20, 40, 5])
    count[table[2, 0].long()] = 3
    parents, fresh = i32([0, 1, 2]), i32(free[:3])
    if kw == "parent":
        parents[1] = 3
    elif kw == "fresh":
        fresh[1] = cache.shape[1]
    elif kw == "taken":
        fresh[1] = table[0, 0]
    elif kw == "taken by many":
        fresh[1] = table[2, 0]
    elif kw == "source":
        fresh[1] = table[1, 2]
    elif kw == "twice":
        fresh[1] = fresh[0]
    elif kw == "page":
        table[1, 1] = -4
    elif kw == "last page":
        table[1, 2] = cache.shape[1]
    else:
        n[1] = 16 * table.shape[1] + 1
    args = (cache, table, n, parents, fresh, count)
    want = [t.clone() for t in args]
    made = [0, 2]
    if kw == "twice":  # one of the two is made
        want_rows = [{0, 2}, {1, 2}]
    else:
        want_rows = [set(made)]
    t, lens = ops.kv_fork(*args)
    assert took_bits() == BAD
    got = {c for c in range(3) if int(lens[c]) > 0}
    assert got in want_rows
    wp = want[3].clone()
    for c in range(3):
        if c not in got:
            wp[c] = -1
    wt, wl = ref.kv_fork(want[0], want[1], want[2], wp, want[4], want[5])
    assert torch.equal(t, wt) and torch.equal(lens, wl)
    assert torch.equal(cache, want[0]) and torch.equal(count, want[5])
    assert torch.equal(table, want[1]) and torch.equal(n, want[2])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("t", [1e37, 1e38, 3e38, 2e-38, 8e-38, 1e-36])
def test_sample_uniform_largest_and_smallest_temperatures(t, dtype):
    """Distances to the maximum, in units of the temperature, whose parts leave fp32's range: the cut of top-p is
    right all the same."""
    g = torch.Generator(device="cuda").manual_seed(11)
    if t > 1:
        logits = (torch.rand(6, 3001, generator=g, device="cuda") * 2 - 1) * 3e38
        logits[:, 7] = 3.2e38
        logits[3] = torch.where(logits[3] > 0, 3e38, -3e38)
    else:
        logits = torch.rand(6, 3001, generator=g, device="cuda") * 12 * t + 2 * t
        logits[3] = torch.where(logits[3] > 8 * t, 10 * t, 6 * t)
    logits = logits.to(dtype)
    u = torch.rand(6, 20, generator=g, device="cuda")
    check_draw(logits, u, [t])
    check_draw(logits, u, [t], top_k=[1, 40, 400, 1000, 2999, 0])
    for p in (0.2, 0.5, 0.9, 0.99):
        check_draw(logits, u, [t], top_p=[p])
        check_draw(logits, u, [t], top_p=[p], top_k=[700])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sample_uniform_nan_settings(dtype):
    nan = float("nan")
    g = torch.Generator(device="cuda").manual_seed(13)
    logits = (torch.randn(4, 3001, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(4, 9, generator=g, device="cuda")
    plain = check_draw(logits, u, [0.8])
    assert torch.equal(check_draw(logits, u, [0.8], top_p=[nan], min_p=[nan]), plain)
    check_draw(logits, u, [0.8], top_k=[30], top_p=[0.7, nan, nan, 0.9], min_p=[nan, 0.1, nan, 0.2])
    check_draw(logits, u, [nan], top_k=[30])


@pytest.mark.parametrize("heads,q_len", [((64, 8, 128), 130), ((8, 8, 64), 1100), ((32, 8, 128), 300)])
def test_many_query_rows(heads, q_len):
    """Prompts behind a shared prefix: query positions by the hundred for each sequence."""
    b = Batch(heads, [2, 1], [100, 33], [q_len, q_len + 7], q_len=q_len)
    b.check(b.run())


# ---------------------------------------------------------------- ids that are not followed
@pytest.mark.parametrize("members", [3, 20, 70])
@pytest.mark.parametrize("where", ["own", "prefix"])
@pytest.mark.parametrize("below", [False, True])
def test_bad_ids_read_page_0(members, where, below):
    """The cache handed over is the middle of a larger one; ids that land in the rest of it are not followed: the
    result is that of page 0 in their place."""
    b = Batch((32, 8, 128), [members], [64], [20])
    front = torch.nan_to_num(b.cache)
    NB = front.shape[1]
    big = torch.full((1, 3 * NB, *front.shape[2:]), 50.0, dtype=front.dtype, device="cuda")
    big[:, NB:2 * NB] = front
    b.cache = big[:, NB:2 * NB]
    assert b.cache.is_contiguous()
    bad = -2 if below else NB + 3
    clean = b.table.clone()
    if where == "own":
        b.table[1, 5] = bad
        clean[1, 5] = 0
    else:  # the prefix is read through the first member's row
        b.table[0, 2] = bad
        clean[:, 2] = 0
    out = b.run()
    assert took_bits() == BAD
    b.table = clean
    b.check(out)


@pytest.mark.parametrize("bad", [-1, 10**6])
def test_kv_free_and_compact_pass_over_bad_ids(bad):
    cache, table, n, count, free = page_state("int8", [40, 20, 100], spare=9)
    want = [t.clone() for t in (cache, table, n, count)]
    table[0, 1] = bad
    keep = int(want[1][0, 1])  # the page that the bad id stands in place of: never given back
    ops.kv_free(table, n, i32([0]), count)
    assert took_bits() == BAD
    want[3][want[1][0, [0, 2]].long()] -= 1
    want[2][0] = 0
    want[1][0, 1] = bad
    assert int(count[keep]) == 1 and torch.equal(count, want[3]) and torch.equal(n, want[2])
    table[1, 0] = bad
    want[1][1, 0] = table[2, 0]  # for the oracle: any held page
    moved, used = ref.kv_compact(*want)
    want[1][1, 0] = bad
    got = ops.kv_compact(cache, table, n, count)
    assert took_bits() == BAD
    assert torch.equal(got[0], moved) and torch.equal(got[1], used)
    for a, w in zip((cache, table, n, count), want):
        assert torch.equal(a, w)


@pytest.mark.parametrize("layers,parents", [(1, [0] * 3000), (33000, [0, 1, -1, 1]), (70, [1] * 40)])
def test_kv_fork_many_children_and_layers(layers, parents):
    """Children by the thousand, and more copy steps of a child than CTAs copy."""
    cache, table, n, count, free = page_state("tiny", [37, 21], spare=len(parents), layers=layers)
    check_fork((cache, table, n, i32(parents), i32(free[:len(parents)]), count))


def test_kv_fork_of_one_fresh_page_by_many_children():
    """One of the children is made, whole, whichever it is; a page that somebody holds is claimed by none."""
    cache, table, n, count, free = page_state("int8", [23 + 16 * (i % 3) for i in range(40)], layers=20)
    held = int(table[7, 0])
    fresh = torch.full((40,), free[0], dtype=torch.int32, device="cuda")
    fresh[30:] = held
    for _ in range(3):
        want, count_want = cache.clone(), count.clone()
        t, lens = ops.kv_fork(cache, table, n, i32(list(range(40))), fresh, count)
        assert took_bits() == BAD
        made = (lens > 0).nonzero()[:, 0].tolist()
        assert len(made) == 1 and made[0] < 30
        parents = i32([c if c in made else -1 for c in range(40)])
        wt, wl = ref.kv_fork(want, table, n, parents, fresh, count_want)
        assert torch.equal(t, wt) and torch.equal(lens, wl) and torch.equal(cache, want)
        assert torch.equal(count, count_want)
        ops.kv_free(t, lens, i32(made), count)
