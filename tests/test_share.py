"""Sequences that share a prompt, without a GPU: plans, and calls that are refused before any launch."""
import pytest
import torch

from bloom_b200 import ops
from bloom_b200.ops import reference as ref


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


# ---------------------------------------------------------------- plans
@pytest.mark.parametrize("sizes,prefix", [([1], [0]), ([4], [512]), ([3, 1, 200], [1000, 0, 77]), ([256], [8192]),
                                          ([1] * 40, [16] * 40), ([300, 2], [31, 100000])])
@pytest.mark.parametrize("heads", [(32, 8, 128, 1), (9, 3, 64, 4), (8, 1, 128, 1)])
def test_plan_covers_every_row_and_key_once(sizes, prefix, heads):
    nq, nkv, D, ql = heads
    p = ops.shared_prefix_plan(sizes, prefix, num_q_heads=nq, num_kv_heads=nkv, head_dim=D, q_len=ql)
    assert p.batch == sum(sizes)
    seen = {}
    for g, r0, s, _ in p.items.tolist():
        first, members, pre, chunk = p.groups[g].tolist()
        assert (first, members, pre) == (sum(sizes[:g]), sizes[g], prefix[g])
        assert s < p.prefix_splits and s * chunk < pre and r0 % p.tile_rows == 0 and r0 < members * ql * (nq // nkv)
        assert (g, r0, s) not in seen
        seen[g, r0, s] = min(chunk, pre - s * chunk)
    splits = [max([s + 1 for (gg, _, s) in seen if gg == g], default=0) for g in range(len(sizes))]
    assert p.seqs.tolist() == [[prefix[g], splits[g]] for g, n in enumerate(sizes) for _ in range(n)]
    for g, (n, pre) in enumerate(zip(sizes, prefix)):
        rows = n * ql * (nq // nkv)
        for r0 in range(0, rows, p.tile_rows):
            assert sum(v for k, v in seen.items() if k[:2] == (g, r0)) == pre
    assert p.suffix_splits in (1, 2, 4, 8)


@pytest.mark.parametrize("kw", [dict(group_sizes=[1, 2], prefix_lens=[3]), dict(group_sizes=[0], prefix_lens=[3]),
                                dict(group_sizes=[2], prefix_lens=[-1]), dict(head_dim=96), dict(num_kv_heads=3),
                                dict(q_len=0)])
def test_plan_refusals(kw):
    args = dict(group_sizes=[2], prefix_lens=[16], num_q_heads=8, num_kv_heads=2, head_dim=64, q_len=1)
    args.update(kw)
    with pytest.raises(ValueError):
        ops.shared_prefix_plan(args.pop("group_sizes"), args.pop("prefix_lens"), **args)


# ---------------------------------------------------------------- refused calls
def shared_args(**kw):
    a = dict(q=torch.zeros(2, 8, 64, dtype=torch.bfloat16),
             kv_cache=torch.zeros(1, 6, 2, 2, 16, 64, dtype=torch.bfloat16), layer=0,
             block_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=i32(20, 20),
             out=torch.zeros(2, 8, 64, dtype=torch.bfloat16),
             plan=ops.shared_prefix_plan([2], [16], num_q_heads=8, num_kv_heads=2, head_dim=64))
    a.update(kw)
    return a


@pytest.mark.parametrize("kw,msg", [
    (dict(q=torch.zeros(2, 8, 64)), "q must be"),
    (dict(q=torch.zeros(2, 8, 65, dtype=torch.bfloat16)[:, :, :64]), "q must be"),
    (dict(q=torch.zeros(8, 2, 64, dtype=torch.bfloat16).transpose(0, 1)), "q must be"),
    (dict(q=torch.zeros(3, 8, 64, dtype=torch.bfloat16), out=torch.zeros(3, 8, 64, dtype=torch.bfloat16)),
     "batch x q_len"),
    (dict(out=torch.zeros(2, 8, 64)), "out must be"),
    (dict(kv_cache=torch.zeros(1, 6, 2 * 2 * 16 * 132, dtype=torch.uint8)), "kv_cache"),
    (dict(kv_cache=torch.zeros(1, 6, 2, 2, 32, 64, dtype=torch.bfloat16)), "kv_cache"),
    (dict(kv_cache=torch.zeros(2, 6, 2, 2, 16, 64, dtype=torch.bfloat16)[:, :3]), "kv_cache"),
    (dict(layer=1), "layer"), (dict(layer=-1), "layer"),
    (dict(block_table=torch.zeros(2, 3, dtype=torch.int64)), "block_table"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), "block_table"),
    (dict(block_table=torch.zeros(3, 2, dtype=torch.int32).t()), "block_table"),
    (dict(seq_lens=torch.zeros(2)), "seq_lens"),
    (dict(seq_lens=i32(1, 1, 1), block_table=torch.zeros(3, 3, dtype=torch.int32),
          q=torch.zeros(3, 8, 64, dtype=torch.bfloat16), out=torch.zeros(3, 8, 64, dtype=torch.bfloat16)),
     "the plan is for another"),
    (dict(plan=ops.shared_prefix_plan([2], [16], num_q_heads=4, num_kv_heads=2, head_dim=64)), "other heads"),
    (dict(plan=ops.shared_prefix_plan([2], [16], num_q_heads=8, num_kv_heads=4, head_dim=64)), "other heads"),
    (dict(), "CUDA device"),
])
def test_shared_prefix_attention_refuses(kw, msg):
    with pytest.raises((RuntimeError, ValueError), match=msg):
        ops.shared_prefix_attention(**shared_args(**kw), scale=1.0)


def fork_args(**kw):
    a = dict(kv_cache=torch.zeros(2, 6, 2, 2, 16, 64, dtype=torch.bfloat16),
             block_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=i32(20, 20), parents=i32(0, 1),
             fresh=i32(4, 5), ref=torch.zeros(6, dtype=torch.int32))
    a.update(kw)
    return a


CACHE_BAD = [(dict(kv_cache=torch.zeros(6, 64)), "kv_cache"),
             (dict(kv_cache=torch.zeros(2, 6, 2, 64)[:, :, 0]), "kv_cache"),
             (dict(kv_cache=torch.zeros(2, 6, 20, dtype=torch.uint8)), "16 bytes"),
             (dict(kv_cache=torch.zeros(12 * 64 + 1)[1:].view(2, 6, 64)), "16-byte"),
             (dict(ref=torch.zeros(5, dtype=torch.int32)), "ref"),
             (dict(ref=torch.zeros(6, dtype=torch.int64)), "ref"),
             (dict(seq_lens=i32(1, 2, 3)), "seq_lens"),
             (dict(block_table=torch.zeros(1, 3, dtype=torch.int32).expand(2, 3)), "block_table"),
             (dict(block_table=torch.zeros(2, 3)), "block_table"), (dict(), "CUDA device")]


@pytest.mark.parametrize("kw,msg", CACHE_BAD + [(dict(parents=i32(0)), "fresh"), (dict(fresh=i32(0)), "fresh"),
                                                (dict(parents=torch.zeros(2)), "parents")])
def test_kv_fork_refuses(kw, msg):
    with pytest.raises(RuntimeError, match=msg):
        ops.kv_fork(**fork_args(**kw))


@pytest.mark.parametrize("kw,msg", CACHE_BAD)
def test_kv_compact_refuses(kw, msg):
    a = fork_args(**kw)
    with pytest.raises(RuntimeError, match=msg):
        ops.kv_compact(a["kv_cache"], a["block_table"], a["seq_lens"], a["ref"])


@pytest.mark.parametrize("kw,msg", [(dict(rows=torch.zeros(2)), "rows"), (dict(seq_lens=i32(1)), "seq_lens"),
                                    (dict(ref=torch.zeros(6)), "ref"), (dict(), "CUDA device")])
def test_kv_free_refuses(kw, msg):
    a = dict(block_table=torch.zeros(2, 3, dtype=torch.int32), seq_lens=i32(3, 3), rows=i32(0),
             ref=torch.zeros(6, dtype=torch.int32))
    a.update(kw)
    with pytest.raises(RuntimeError, match=msg):
        ops.kv_free(**a)


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=torch.zeros(2, 10, dtype=torch.float16)), "logits"),
    (dict(logits=torch.zeros(10, 2).t()), "logits"),
    (dict(logits=torch.zeros(2, 0)), "tokens per row"),
    (dict(logits=torch.zeros(1, 1).expand(2, (1 << 18) + 1)), "logits|tokens per row"),
    (dict(u=torch.zeros(3)), "u must be"), (dict(u=torch.zeros(2, dtype=torch.float64)), "u must be"),
    (dict(u=torch.zeros(3, 2).t()), "u must be"),
    (dict(out=torch.zeros(2, 1, dtype=torch.int32)), "out must be"),
    (dict(out=torch.zeros(2, dtype=torch.int64)), "out must be"),
    (dict(temperature=torch.ones(1)), "temperature"), (dict(top_k=torch.ones(2)), "top_k"),
    (dict(top_p=torch.ones(2, dtype=torch.float64)), "top_p"), (dict(min_p=torch.ones(2, 1)), "min_p"),
    (dict(), "CUDA device"),
])
def test_sample_uniform_refuses(kw, msg):
    a = dict(logits=torch.zeros(2, 10), u=torch.zeros(2), temperature=torch.ones(2))
    a.update(kw)
    with pytest.raises(RuntimeError, match=msg):
        ops.sample_uniform(**a)


# ---------------------------------------------------------------- the oracles themselves, on cases worked out by hand
def test_oracle_draw():
    logits = torch.log(torch.tensor([[4.0, 2.0, 1.0, 1.0]]))
    one = torch.ones(1)
    u = torch.tensor([[0.0, 0.4, 0.6, 0.8, 0.95]])
    assert ref.sample_uniform(logits, u, one).tolist() == [[0, 0, 1, 2, 3]]
    assert ref.sample_uniform(logits, u, one, top_k=i32(3)).tolist() == [[0, 0, 1, 1, 2]]  # of 7: 4, 6
    assert ref.sample_uniform(logits, u, one, top_p=torch.tensor([0.7])).tolist() == [[0, 0, 0, 1, 1]]
    assert ref.sample_uniform(logits, u, one, min_p=torch.tensor([0.4])).tolist() == [[0, 0, 0, 1, 1]]
    assert ref.sample_uniform(logits, u, torch.zeros(1)).tolist() == [[0] * 5]
    assert ref.sample_uniform(torch.full((1, 3), float("-inf")), u, one).tolist() == [[-1] * 5]


def test_oracle_pages():
    cache = torch.arange(6.0).view(1, 6, 1).clone()
    table, lens, count = torch.tensor([[3, 1], [5, 0]], dtype=torch.int32), i32(20, 16), i32(0, 1, 0, 1, 0, 1)
    t, n = ref.kv_fork(cache, table, lens, i32(0, 1, -1), i32(2, 0, 0), count)
    assert t.tolist() == [[3, 2], [5, 0], [0, 0]] and n.tolist() == [20, 16, 0]
    assert count.tolist() == [0, 1, 1, 2, 0, 2] and cache[0, 2, 0] == 1
    ref.kv_free(table, lens, i32(0, 0), count)
    assert count.tolist() == [0, 0, 1, 1, 0, 2] and lens.tolist() == [0, 16]
    moved, used = ref.kv_compact(cache, t, n, count)
    assert used.tolist() == [3] and moved.tolist() == [-1, -1, 2, 0, -1, 1]
    assert t.tolist() == [[0, 2], [1, 0], [0, 0]] and count.tolist() == [1, 2, 1, 0, 0, 0]
    assert cache[0, :3, 0].tolist() == [3, 5, 1]


def test_oracle_draw_with_nan_settings():
    """NaN is in no range that a setting is on in: off, and a NaN temperature is greedy."""
    nan = torch.tensor([float("nan")])
    logits = torch.log(torch.tensor([[2.0, 4.0, 1.0, 1.0]]))
    u = torch.tensor([[0.0, 0.4, 0.6, 0.8, 0.95]])
    plain = ref.sample_uniform(logits, u, torch.ones(1)).tolist()
    assert plain == [[0, 1, 1, 2, 3]]
    assert ref.sample_uniform(logits, u, torch.ones(1), min_p=nan).tolist() == plain
    assert ref.sample_uniform(logits, u, torch.ones(1), top_p=nan).tolist() == plain
    assert ref.sample_uniform(logits, u, nan).tolist() == [[1] * 5]


@pytest.mark.parametrize("scale", [float("nan"), float("inf"), float("-inf"), 3e38])
def test_shared_prefix_attention_refuses_scales(scale):
    with pytest.raises(RuntimeError, match="scale must be"):
        ops.shared_prefix_attention(**shared_args(), scale=scale)


@pytest.mark.parametrize("q_len,msg", [(128, "CUDA device"), (1 << 14, "CUDA device"), (1 << 16, "too many heads")])
def test_shared_prefix_attention_query_rows(q_len, msg):
    """As many query rows as the grid holds: KV heads x chunks of 32 rows up to 65,535."""
    nq, nkv = 64, 32
    q = torch.zeros(1, nq, 64, dtype=torch.bfloat16).expand(q_len, nq, 64)
    a = shared_args(q=q, out=torch.empty(q_len, nq, 64, dtype=torch.bfloat16), seq_lens=i32(20),
                    kv_cache=torch.zeros(1, 6, 2, nkv, 16, 64, dtype=torch.bfloat16),
                    block_table=torch.zeros(1, 3, dtype=torch.int32),
                    plan=ops.shared_prefix_plan([1], [16], num_q_heads=nq, num_kv_heads=nkv, head_dim=64, q_len=q_len))
    with pytest.raises(RuntimeError, match=msg):
        ops.shared_prefix_attention(**a, scale=1.0)
