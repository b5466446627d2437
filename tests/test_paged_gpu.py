"""The paged key/value cache operators against plain 64-bit forms: the page write, the attention of one new token
and the causal attention of packed prompts, alone, together and in captured graphs."""
import pytest
import torch

from tests.paged_reference import BF16, Case, assert_within, attend, rng, tables, turn

pytestmark = pytest.mark.gpu

# q heads, kv heads, head dim: the talker's, the codec transformer's, and groups of 1, 3, 4, 7, 8, 9 and 16
GEOMETRIES = [(16, 8, 128), (8, 8, 64), (12, 4, 64), (8, 2, 128), (14, 2, 64), (8, 1, 128), (9, 1, 128), (16, 1, 64)]
PAGES = [16, 48, 64, 256]


@pytest.fixture(scope="module")
def ops(cuda):
    from qwen3_tts_b200 import ops as _ops
    return _ops


def rows_of(shape, seed, strided):
    rows, width = shape[0], shape[1] * shape[2] if len(shape) == 3 else shape[1]
    x = torch.randn(rows, width + (40 if strided else 0), generator=rng(seed)).to(BF16)
    return x[:, :width].unflatten(1, shape[1:]) if len(shape) == 3 else x[:, :width]


def on(x, device):
    """x on the device, its strides kept."""
    if x.is_contiguous():
        return x.to(device)
    whole = torch.as_strided(x, (x.shape[0], x.stride(0)), (x.stride(0), 1))
    return torch.as_strided(whole.to(device), x.shape, x.stride())


# ------------------------------------------------------------------ the write
def check_write(ops, cuda, q, kv, d, page, lengths, *, new, norm, strided, one_pool=False, seed=0):
    case = Case(lengths, kv, d, page, seed=seed, one_pool=one_pool)
    if new:   # the last position of every sequence
        at, seq = torch.tensor(lengths) - 1, None
    else:     # every position of every sequence, in a shuffled order
        at = torch.cat([torch.arange(n) for n in lengths])
        seq = torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths))
        order = torch.randperm(len(at), generator=rng(seed + 1))
        at, seq = at[order], seq[order]
    rows = len(at)
    qkv = rows_of((rows, (q + 2 * kv) * d), seed + 2, strided)
    weights = [(1 + 0.2 * torch.randn(d, generator=rng(seed + 3 + i))).to(BF16) if norm else None for i in range(2)]
    cos, sin = tables(max(lengths) + 5, d)
    rotary = at + 4
    keys, values, table = case.to(cuda)
    dev = [None if t is None else t.to(cuda) for t in (*weights, cos, sin, rotary, at, seq)]
    got = ops.paged_qk_norm_rope_kv(on(qkv, cuda), dev[0], dev[1], 1e-6, dev[2], dev[3], dev[4], dev[5], table, keys,
                                    values, q_heads=q, kv_heads=kv, head_dim=d, sequences=dev[6])
    assert ops.read_status(cuda) == 0
    x = qkv.reshape(rows, q + 2 * kv, d)
    want, bound = turn(x[:, :q], weights[0], cos[rotary], sin[rotary], 1e-6)
    assert_within(got, want, bound, "queries")
    want, bound = turn(x[:, q:q + kv], weights[1], cos[rotary], sin[rotary], 1e-6)
    where = case.table[torch.arange(rows) if seq is None else seq, at // page].long()
    assert_within(keys.cpu()[where, :, at % page], want, bound, "keys")
    assert torch.equal(values.cpu()[where, :, at % page], x[:, q + kv:])
    for pool, before in ((keys.cpu(), case.keys.clone()), (values.cpu(), case.values.clone())):
        pool[where, :, at % page] = 0
        before[where, :, at % page] = 0
        assert torch.equal(pool.view(torch.int16), before.view(torch.int16))  # nothing else is touched


@pytest.mark.parametrize("q,kv,d", GEOMETRIES)
@pytest.mark.parametrize("new", [True, False])
def test_write_heads(ops, cuda, q, kv, d, new):
    check_write(ops, cuda, q, kv, d, 32, [1, 31, 32, 33, 70], new=new, norm=True, strided=False)


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("norm,strided,one_pool", [(True, True, False), (False, False, True), (False, True, True)])
def test_write_pages_strides_and_rows_without_norm(ops, cuda, page, norm, strided, one_pool):
    check_write(ops, cuda, 16, 8, 128, page, [5, 17, page, page + 1, 3 * page], new=False, norm=norm, strided=strided,
                one_pool=one_pool)


@pytest.mark.parametrize("q,kv,d,norm", [(16, 8, 128, True), (8, 8, 64, False), (14, 2, 64, True), (9, 1, 128, True)])
def test_write_many_rows(ops, cuda, q, kv, d, norm):
    check_write(ops, cuda, q, kv, d, 64, [1001, 3, 900], new=False, norm=norm, strided=True)


@pytest.mark.parametrize("count", [1, 2, 64, 257])
def test_write_step_batches(ops, cuda, count):
    check_write(ops, cuda, 16, 8, 128, 16, [1 + 7 * i % 60 for i in range(count)], new=True, norm=True, strided=False,
                seed=count)


def write_args(ops, cuda, rows=3, q=4, kv=2, d=64, page=16, columns=2):
    table = torch.arange(rows * columns, dtype=torch.int32, device=cuda).view(rows, columns)
    cos, sin = (t.to(cuda) for t in tables(64, d))
    qkv = torch.randn(rows, (q + 2 * kv) * d, generator=rng(9)).to(BF16).to(cuda)
    pool = [torch.zeros(rows * columns, kv, page, d, dtype=BF16, device=cuda) for _ in range(2)]
    return qkv, cos, sin, table, pool


def test_write_skips_padding_rows_and_flags_bad_positions(ops, cuda):
    qkv, cos, sin, table, (keys, values) = write_args(ops, cuda)
    out = torch.full((3, 4, 64), 7.0, dtype=BF16, device=cuda)

    def write(at, sequences, rotary=(1, 1, 1), page_table=table):
        keys.zero_(), values.zero_(), out.fill_(7.0)
        ops.paged_qk_norm_rope_kv(qkv, None, None, 1e-6, cos, sin, torch.tensor(rotary, device=cuda),
                                  torch.tensor(at, device=cuda), page_table, keys, values, q_heads=4, kv_heads=2,
                                  head_dim=64, sequences=torch.tensor(sequences, device=cuda), query_out=out)
        written = values.ne(0).any(-1).any(1).nonzero().tolist()
        return written, out.ne(7.0).flatten(1).any(1).tolist(), ops.read_status(cuda)

    assert write((3, 4, 5), (0, -1, 2)) == ([[0, 3], [4, 5]], [True, False, True], 0)
    assert write((3, 1 << 40, 5), (0, -(1 << 60), 2), rotary=(1, -5, 1)) == ([[0, 3], [4, 5]], [True, False, True], 0)
    assert write((3, 32, 5), (0, 1, 2)) == ([[0, 3], [4, 5]], [True] * 3, 8)      # past the table's columns
    assert write((3, -1, 5), (0, 1, 2)) == ([[0, 3], [4, 5]], [True] * 3, 8)
    assert write((3, 4, 5), (0, 3, 2)) == ([[0, 3], [4, 5]], [True] * 3, 8)       # past the table's rows
    assert write((3, 4, 5), (0, 1, 2), rotary=(1, 64, 1)) == ([[0, 3], [2, 4], [4, 5]], [True] * 3, 8)
    bad = table.clone()
    bad[1, 0] = 6
    assert write((3, 4, 5), (0, 1, 2), page_table=bad) == ([[0, 3], [4, 5]], [True] * 3, 8)
    bad[1, 0] = -1
    assert write((3, 20, 5), (0, 1, 2), page_table=bad) == ([[0, 3], [3, 4], [4, 5]], [True] * 3, 0)


# ------------------------------------------------------------------ one new token
def check_decode(ops, cuda, q, kv, d, page, lengths, *, strided=False, one_pool=False, seed=0, scale=None, context=None,
                 columns=None, share=0, gain=1.0):
    case = Case(lengths, kv, d, page, seed=seed, one_pool=one_pool, columns=columns, share=share)
    query = (gain * rows_of((len(lengths), q, d), seed + 1, strided)) if not strided else \
        rows_of((len(lengths), q, d), seed + 1, strided)
    keys, values, table = case.to(cuda)
    got = ops.paged_decode_attention(on(query, cuda), keys, values, table, (torch.tensor(lengths) - 1).to(cuda),
                                     scale=scale, context=context)
    assert ops.read_status(cuda) == 0
    for r, n in enumerate(lengths):
        want, bound = attend(query[r], *case.sequence(r, n), d ** -0.5 if scale is None else scale)
        assert_within(got[r], want, bound, f"row {r} of {n} keys")


# The table's capacity is all that a call knows of the lengths beforehand: one that could hold very long contexts
# makes it cut the keys of all rows into even ranges instead of going row by row.
BOTH = pytest.mark.parametrize("capacity", [None, 1 << 17], ids=["rows", "ranges"])


def columns_for(capacity, page):
    return None if capacity is None else capacity // page


@BOTH
@pytest.mark.parametrize("q,kv,d", GEOMETRIES)
def test_decode_heads(ops, cuda, q, kv, d, capacity):
    check_decode(ops, cuda, q, kv, d, 32, [1, 0, 15, 16, 17, 31, 32, 33, 127, 128, 129, 400],
                 columns=columns_for(capacity, 32))


@BOTH
@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("strided,one_pool", [(True, False), (False, True)])
def test_decode_pages_and_strides(ops, cuda, page, strided, one_pool, capacity):
    check_decode(ops, cuda, 16, 8, 128, page, [page - 1, page, page + 1, 5 * page + 3], strided=strided,
                 one_pool=one_pool, columns=columns_for(capacity, page) or 9)


@pytest.mark.parametrize("lengths", [[1], [0], [0, 0, 0], [4097], [1, 8000, 1], [3000] + [5] * 40, [513] * 70])
@pytest.mark.parametrize("q,kv,d", [(16, 8, 128), (16, 1, 64)])
@BOTH
def test_decode_lengths(ops, cuda, lengths, q, kv, d, capacity):
    check_decode(ops, cuda, q, kv, d, 64, lengths, columns=columns_for(capacity, 64))


def test_decode_long_context(ops, cuda):
    check_decode(ops, cuda, 8, 2, 128, 128, [70001, 1, 33333])


@BOTH
@pytest.mark.parametrize("count", [30, 300, 1500, 4097])
def test_decode_many_rows(ops, cuda, count, capacity):
    check_decode(ops, cuda, 4, 2, 64, 16, [(37 * i) % 90 for i in range(count)], seed=count,
                 columns=columns_for(capacity, 16))


def test_decode_context_bound_shared_pages_and_scale(ops, cuda):
    check_decode(ops, cuda, 16, 8, 128, 16, [90, 41, 64, 3], share=2, context=90, columns=40)
    check_decode(ops, cuda, 16, 8, 128, 16, [90, 41, 64, 3], scale=0.5)       # peaked weights
    check_decode(ops, cuda, 16, 8, 128, 16, [90, 41, 64, 3], scale=-0.25)
    check_decode(ops, cuda, 16, 8, 128, 16, [90, 41, 64, 3], scale=0.0)


@BOTH
def test_decode_rising_scores_move_the_reference(ops, cuda, capacity):
    """Scores that grow by far more than the lazy margin from step to step, up and down again."""
    n, d = 300, 64
    case = Case([n], 1, d, 16, columns=columns_for(capacity, 16))
    keys, _ = case.sequence(0, n)
    ramp = torch.cat((torch.arange(200.0), torch.arange(100.0).flip(0)))
    for j in range(n):
        case.keys[case.table[0, j // 16], 0, j % 16] = torch.full((d,), ramp[j].item() / 8).to(BF16)
    query = torch.ones(1, 2, d, dtype=BF16)
    query[0, 1] = -1
    k, v, table = case.to(cuda)
    got = ops.paged_decode_attention(query.to(cuda), k, v, table, torch.tensor([n - 1], device=cuda))
    want, bound = attend(query[0], *case.sequence(0, n), d ** -0.5)
    assert_within(got[0], want, bound)


@BOTH
def test_decode_infinite_scores_follow_the_formula(ops, cuda, capacity):
    """A key of -inf has weight 0 wherever it stands; only -inf scores, or one of +inf, have no value."""
    n, d = 40, 64
    for where in (0, 5, 39):
        case = Case([n], 1, d, 16, columns=columns_for(capacity, 16))
        case.keys[case.table[0, where // 16], 0, where % 16, 0] = -float("inf")
        query = torch.ones(1, 1, d, dtype=BF16)
        k, v, table = case.to(cuda)
        got = ops.paged_decode_attention(query.to(cuda), k, v, table, torch.tensor([n - 1], device=cuda))
        rest = [j for j in range(n) if j != where]
        keys, values = case.sequence(0, n)
        want, bound = attend(query[0], keys[:, rest], values[:, rest], d ** -0.5)
        assert_within(got[0], want, bound)
        got = ops.paged_decode_attention(-query.to(cuda), k, v, table, torch.tensor([n - 1], device=cuda))
        assert got.isnan().all()
    case.keys[..., 0] = -float("inf")
    k, v, table = case.to(cuda)
    got = ops.paged_decode_attention(query.to(cuda), k, v, table, torch.tensor([n - 1], device=cuda))
    assert got.isnan().all()


@BOTH
def test_decode_flags_bad_positions_and_pages(ops, cuda, capacity):
    """The row with the bad index is unspecified; its neighbours are right and nothing faults."""
    lengths = [40, 40, 40]
    case = Case(lengths, 8, 128, 16, columns=columns_for(capacity, 16))
    query = rows_of((3, 16, 128), 1, False)
    keys, values, table = case.to(cuda)

    def decode(positions, page_table=table):
        got = ops.paged_decode_attention(query.to(cuda), keys, values, page_table, torch.tensor(positions, device=cuda))
        for r in (0, 2):
            assert_within(got[r], *attend(query[r], *case.sequence(r, 40), 128 ** -0.5))
        return ops.read_status(cuda)

    assert decode((39, 39, 39)) == 0
    assert decode((39, -2, 39)) == 8
    for entry in (len(case.keys), -1, -(1 << 31), (1 << 31) - 1):
        bad = table.clone()
        bad[1, 1] = entry
        assert decode((39, 39, 39), bad) == 8
        assert decode((39, 15, 39), bad) == 0  # the entry is not needed


def test_decode_clamps_a_position_past_the_context(ops, cuda):
    case = Case([64, 64], 8, 128, 16, columns=9)
    query = rows_of((2, 16, 128), 1, False)
    keys, values, table = case.to(cuda)
    got = ops.paged_decode_attention(query.to(cuda), keys, values, table, torch.tensor([64, 20], device=cuda), context=64)
    assert ops.read_status(cuda) == 8
    assert_within(got[0], *attend(query[0], *case.sequence(0, 64), 128 ** -0.5))
    assert_within(got[1], *attend(query[1], *case.sequence(1, 21), 128 ** -0.5))


@BOTH
def test_decode_repeats_bit_for_bit(ops, cuda, capacity):
    case = Case([5000, 77, 1234, 1], 8, 128, 64, columns=columns_for(capacity, 64))
    query = rows_of((4, 16, 128), 1, False).to(cuda)
    keys, values, table = case.to(cuda)
    at = torch.tensor([4999, 76, 1233, 0], device=cuda)
    first = ops.paged_decode_attention(query, keys, values, table, at)
    for _ in range(20):
        assert torch.equal(ops.paged_decode_attention(query, keys, values, table, at), first)


# ------------------------------------------------------------------ packed prompts
def check_prompt(ops, cuda, q, kv, d, page, counts, starts, *, lead=0, tail=0, strided=False, one_pool=False, seed=0,
                 scale=None, columns=None):
    lengths = [max(0, n + s) if n else max(0, s) for n, s in zip(counts, starts)]
    case = Case(lengths, kv, d, page, seed=seed, one_pool=one_pool, columns=columns)
    rows = lead + sum(counts) + tail
    query = rows_of((rows, q, d), seed + 1, strided)
    offsets = torch.tensor([lead + sum(counts[:i]) for i in range(len(counts) + 1)])
    keys, values, table = case.to(cuda)
    out = torch.full((rows, q, d), 5.0, dtype=BF16, device=cuda)
    got = ops.paged_prefill_attention(on(query, cuda), keys, values, table, offsets.to(cuda),
                                      torch.tensor(starts).to(cuda), out=out, scale=scale)
    assert ops.read_status(cuda) == 0
    assert (got[:lead] == 5).all() and (got[rows - tail:] == 5).all()
    scale = d ** -0.5 if scale is None else scale
    for s, n in enumerate(counts):
        for i in range(n):
            r, seen = int(offsets[s]) + i, max(0, starts[s] + i + 1)
            if n > 300 and i % 37 and i < n - 3:
                continue
            want, bound = attend(query[r], *case.sequence(s, seen), scale)
            assert_within(got[r], want, bound, f"sequence {s} row {i} of {seen} keys")


@pytest.mark.parametrize("q,kv,d", GEOMETRIES)
def test_prompt_heads(ops, cuda, q, kv, d):
    check_prompt(ops, cuda, q, kv, d, 32, [1, 33, 70, 5], [0, 0, 0, 0])


@pytest.mark.parametrize("page", PAGES)
@pytest.mark.parametrize("strided,one_pool", [(True, False), (False, True)])
def test_prompt_pages_and_strides(ops, cuda, page, strided, one_pool):
    check_prompt(ops, cuda, 16, 8, 128, page, [129, 1, 64, 200], [0, 31, 0, 5], strided=strided, one_pool=one_pool,
                 columns=20)


@pytest.mark.parametrize("counts,starts", [([1], [0]), ([127], [0]), ([128], [0]), ([129], [0]), ([257], [0]),
                                           ([1, 1, 1], [0, 500, 129]), ([0, 5, 0, 0, 3, 0], [0, 0, 7, 0, 300, 0]),
                                           ([40, 90], [1000, 64]), ([30, 6], [-7, -6]), ([3], [-5]), ([0], [0])])
@pytest.mark.parametrize("q,kv,d", [(16, 8, 128), (8, 8, 64), (8, 1, 128)])
def test_prompt_lengths_and_prefixes(ops, cuda, counts, starts, q, kv, d):
    check_prompt(ops, cuda, q, kv, d, 64, counts, starts, lead=2, tail=3)


def test_prompt_long(ops, cuda):
    check_prompt(ops, cuda, 4, 1, 128, 64, [1500, 700], [0, 2000])
    check_prompt(ops, cuda, 2, 2, 64, 16, [1500], [0], strided=True)


@pytest.mark.parametrize("counts,starts", [([1], [5000]), ([90, 3], [3000, 0]), ([64, 1, 500], [4000, 9000, 0]),
                                           ([40] * 9, [700] * 9), ([33], [-20]), ([20], [-40]),
                                           ([2000, 1, 300, 0, 1111], [0, 3, 2000, 5, 77])])
@pytest.mark.parametrize("q,kv,d,page", [(16, 8, 128, 64), (8, 8, 64, 16), (16, 1, 128, 48), (6, 1, 64, 256)])
def test_prompt_ranges(ops, cuda, counts, starts, q, kv, d, page):
    """Tables that could hold long contexts: the key tiles of all items in even ranges, some items in parts."""
    check_prompt(ops, cuda, q, kv, d, page, counts, starts, columns=(1 << 17) // page + 1, lead=1, tail=1)


def test_prompt_wide_groups(ops, cuda):
    check_prompt(ops, cuda, 70, 1, 64, 16, [5, 40], [0, 3])
    check_prompt(ops, cuda, 70, 1, 64, 16, [5, 40], [0, 3], columns=1000)


@pytest.mark.parametrize("count", [31, 32, 33, 1024, 1500, 2048, 2049])
def test_prompt_many_sequences(ops, cuda, count):
    counts, starts = [(7 * i) % 4 for i in range(count)], [(5 * i) % 23 for i in range(count)]
    check_prompt(ops, cuda, 4, 2, 128, 16, counts, starts)
    if count <= 33:
        check_prompt(ops, cuda, 4, 2, 128, 16, [5 * n for n in counts], [90 * n for n in starts], columns=1 << 13)


def test_prompt_sequences_of_many_lengths(ops, cuda):
    """Lengths around every multiple of a tile pair's positions, in an order that puts them at every offset."""
    counts = [n + d for n in (128, 256, 384) for d in (-1, 0, 1)] + [1] * 40 + [127, 129, 255]
    check_prompt(ops, cuda, 4, 2, 64, 16, counts, [0] * len(counts))
    check_prompt(ops, cuda, 4, 2, 64, 16, counts[::-1], [0] * len(counts), columns=1 << 13, lead=3)
    check_prompt(ops, cuda, 4, 2, 128, 16, [(13 * i) % 41 for i in range(120)], [(5 * i) % 23 for i in range(120)])


@pytest.mark.parametrize("q,kv,d", [g for g in GEOMETRIES if g[1] < 8])
def test_prompt_heads_in_tiles(ops, cuda, q, kv, d):
    check_prompt(ops, cuda, q, kv, d, 32, [1, 33, 470, 5], [0, 0, 0, 40], lead=1, tail=2)


def test_prompt_wide_groups_in_tiles(ops, cuda):
    check_prompt(ops, cuda, 70, 1, 64, 16, [5, 140], [0, 3])


# few rows: one CTA, or a cluster, for each row and KV head
@pytest.mark.parametrize("counts,starts", [([1], [5000]), ([1], [0]), ([2], [700]), ([4], [4000]), ([9], [-4]), ([18], [120]),
                                           ([3, 0, 1], [2000, 0, 100]), ([1] * 9, [513] * 9), ([0, 0, 5, 0], [0, 3, 60, 0]),
                                           ([48], [0]), ([20, 30], [100, 9])])
@pytest.mark.parametrize("q,kv,d,page", [(16, 8, 128, 64), (8, 8, 64, 16), (16, 1, 128, 48), (9, 1, 64, 256)])
def test_prompt_of_few_rows(ops, cuda, counts, starts, q, kv, d, page):
    check_prompt(ops, cuda, q, kv, d, page, counts, starts, lead=2, tail=1, strided=True)


@pytest.mark.parametrize("group", [1, 2, 3, 4, 5, 6, 7, 8, 9])
@pytest.mark.parametrize("kv,d", [(2, 64), (1, 128)])
def test_prompt_rows_that_share_their_keys(ops, cuda, group, kv, d):
    """Tables of more than 768 positions: 8 / group consecutive rows of a sequence make one item."""
    check_prompt(ops, cuda, group * kv, kv, d, 16, [1, 7, 8, 9, 0, 17], [1000, 41, 0, 1009, 5, 333], lead=1, tail=2, strided=True)
    check_prompt(ops, cuda, group * kv, kv, d, 16, [9, 12, 3], [-3, -20, 12], columns=64)   # padding inside of an item


@pytest.mark.parametrize("count", [31, 33, 64, 127, 128, 129, 300])
def test_prompt_of_few_rows_among_many_sequences(ops, cuda, count):
    counts, starts = [int(i % 3 == 1) + int(i == count - 1) for i in range(count)], [(7 * i) % 90 for i in range(count)]
    check_prompt(ops, cuda, 4, 2, 128, 16, counts, starts, lead=1, tail=2)


@pytest.mark.parametrize("rows,ranks", [(1, 8), (3, 4), (9, 2), (18, 1)])
@pytest.mark.parametrize("past", [0, 1])
def test_prompt_on_either_side_of_the_limit_for_rows(ops, cuda, rows, ranks, past):
    """16 query and 8 KV heads: by rows up to 6144 keys a CTA of the table, in tiles past them; the same results."""
    check_prompt(ops, cuda, 16, 8, 128, 64, [rows], [1500], columns=6144 * ranks // 64 + past)


def test_prompts_of_few_rows_with_odd_offsets_are_flagged(ops, cuda):
    case = Case([8, 8, 8], 2, 64, 16)
    query = rows_of((12, 4, 64), 1, False)
    keys, values, table = case.to(cuda)

    def prompt(offsets, page_table):
        out = torch.full_like(query, 5.0, device=cuda)
        ops.paged_prefill_attention(query.to(cuda), keys, values, page_table, torch.tensor(offsets, device=cuda),
                                    torch.zeros(len(offsets) - 1, dtype=torch.int64, device=cuda), out=out)
        return out, ops.read_status(cuda)

    for offsets in ([0, 4, 8, 13], [-1, 4, 8, 12], [0, 6, 3, 9], [0, 2 ** 40, 8, 12]):
        out, status = prompt(offsets, table)
        assert status == 8
        owners = [s for s in range(3) if 0 <= offsets[s] < offsets[s + 1] <= 12]
        for r in range(12):
            mine = [s for s in owners if offsets[s] <= r < offsets[s + 1]]
            near = [(out[r].double().cpu() - want).abs() <= bound for want, bound in
                    (attend(query[r], *case.sequence(s, r - offsets[s] + 1), 0.125) for s in mine)]
            assert torch.stack(near).any(0).all() if mine else (out[r] == 5).all(), f"{offsets} row {r}"
    many = [0, 4] + [8] * 149   # past the sequences that one look takes
    assert prompt(many, table.repeat(50, 1))[1] == 0
    for at, value in ((1, -3), (0, -1), (70, 13), (150, 13), (149, 0)):
        out, status = prompt(many[:at] + [value] + many[at + 1:], table.repeat(50, 1))
        assert status == 8 and (out[8:] == 5).all()


def test_prompts_of_few_rows_repeat_captured_and_in_clusters(ops, cuda):
    case = Case([3003, 2002], 8, 128, 64)
    query = rows_of((5, 16, 128), 1, False).to(cuda)
    keys, values, table = case.to(cuda)
    offsets, starts = torch.tensor([0, 3, 5], device=cuda), torch.tensor([3000, 2000], device=cuda)
    out = torch.empty_like(query)
    want = ops.paged_prefill_attention(query, keys, values, table, offsets, starts, out=out).clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_prefill_attention(query, keys, values, table, offsets, starts, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    # the same keys one new token at a time
    for r, s in enumerate((0, 0, 0, 1, 1)):
        at = starts[s:s + 1] + (r - int(offsets[s]))
        alone = ops.paged_decode_attention(query[r:r + 1], keys, values, table[s:s + 1], at)
        wanted, bound = attend(query[r].cpu(), *case.sequence(s, int(at) + 1), 128 ** -0.5)
        assert_within(alone[0], wanted, bound, f"row {r} alone")
        assert_within(want[r], wanted, bound, f"row {r}")


def test_prompt_scale(ops, cuda):
    check_prompt(ops, cuda, 16, 8, 128, 16, [150], [0], scale=0.5)
    check_prompt(ops, cuda, 16, 8, 128, 16, [150], [0], scale=-0.25)


def test_prompt_flags_bad_pages(ops, cuda):
    case = Case([40, 40, 40], 8, 128, 16)
    query = rows_of((120, 16, 128), 1, False)
    keys, values, table = case.to(cuda)
    offsets, starts = torch.tensor([0, 40, 80, 120], device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)

    def prompt(page_table, start=starts):
        got = ops.paged_prefill_attention(query.to(cuda), keys, values, page_table, offsets, start,
                                          out=torch.zeros_like(query, device=cuda))
        for r in list(range(40)) + list(range(80, 120)):
            want, bound = attend(query[r], *case.sequence(r // 40, r % 40 + 1), 128 ** -0.5)
            assert_within(got[r], want, bound, f"row {r}")
        return ops.read_status(cuda)

    assert prompt(table) == 0
    for entry in (len(case.keys), -1, (1 << 31) - 1):
        bad = table.clone()
        bad[1, 1] = entry
        assert prompt(bad) == 8
    # a start that puts the rows past what the table can hold
    assert prompt(table, torch.tensor([0, 20, 0], device=cuda)) == 8


# ------------------------------------------------------------------ together
def serve(ops, cuda, steps, capture):
    """A prompt of three sequences, then `steps` decode steps, all through the pages; (outputs, their checks)."""
    q, kv, d, page = 16, 8, 128, 16
    counts = [37, 5, 64]
    case = Case([n + steps for n in counts], kv, d, page, seed=4)
    case.keys.fill_(float("nan")), case.values.fill_(float("nan"))
    keys, values, table = case.to(cuda)
    cos, sin = tables(128, d)
    weights = [(1 + 0.2 * torch.randn(d, generator=rng(50 + i))).to(BF16) for i in range(2)]
    dev = [t.to(cuda) for t in (*weights, cos, sin)]
    rows = sum(counts)
    qkv = torch.randn(rows + 3 * steps, (q + 2 * kv) * d, generator=rng(6)).to(BF16)
    prompt, new = qkv[:rows].to(cuda), qkv[rows:].view(steps, 3, -1).to(cuda)
    at = torch.cat([torch.arange(n) for n in counts]).to(cuda)
    seq = torch.repeat_interleave(torch.arange(3), torch.tensor(counts)).to(cuda)
    offsets = torch.tensor([0, 37, 42, 106], device=cuda)
    heads = dict(q_heads=q, kv_heads=kv, head_dim=d)
    queries = ops.paged_qk_norm_rope_kv(prompt, dev[0], dev[1], 1e-6, dev[2], dev[3], at, at, table, keys, values,
                                        sequences=seq, **heads)
    outs = [ops.paged_prefill_attention(queries, keys, values, table, offsets,
                                        torch.zeros(3, dtype=torch.int64, device=cuda),
                                        out=torch.empty_like(queries))]
    positions, row = torch.tensor(counts, device=cuda), torch.empty_like(new[0])
    out = torch.empty(3, q, d, dtype=BF16, device=cuda)

    def step():
        query = ops.paged_qk_norm_rope_kv(row, dev[0], dev[1], 1e-6, dev[2], dev[3], positions, positions, table, keys,
                                          values, **heads)
        ops.paged_decode_attention(query, keys, values, table, positions, out=out)
        ops.advance(positions)

    if capture:
        row.copy_(new[0])
        saved = positions.clone()
        step()
        positions.copy_(saved)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        positions.copy_(saved)
    for i in range(steps):
        row.copy_(new[i])
        graph.replay() if capture else step()
        outs.append(out.clone())
    assert ops.read_status(cuda) == 0
    return outs, (counts, qkv, weights, cos, sin)


def check_served(outs, inputs, steps):
    """Attention over the bf16 queries, keys and values of the write's own formula, in 64 bits. Where such a value lies
    at a rounding boundary the kernel's may be one step off, so each score may move by 2^-7 of scale * sum |q k| twice."""
    counts, qkv, weights, cos, sin = inputs
    q, kv, d = 16, 8, 128
    rows = sum(counts)
    for s, n in enumerate(counts):
        mine = torch.cat((qkv[sum(counts[:s]):sum(counts[:s]) + n], qkv[rows:].view(steps, 3, -1)[:, s]))
        at = torch.arange(n + steps)
        x = mine.view(-1, q + 2 * kv, d)
        queries, keys = (turn(x[:, a:b], w, cos[at], sin[at], 1e-6)[0].to(BF16)
                         for a, b, w in ((0, q, weights[0]), (q, q + kv, weights[1])))
        values = x[:, q + kv:].double().transpose(0, 1)
        for i in range(n + steps):
            k, v = keys[:i + 1].double().transpose(0, 1), values[:, :i + 1]
            want, bound = attend(queries[i], k, v, d ** -0.5)
            got = outs[0][sum(counts[:s]) + i] if i < n else outs[1 + i - n][s]
            # steps of a value at a boundary are rare: 1 element in 2^12 (fp32 error over a bf16 step), so at most a
            # few of the 128 products of a score move, each by 2^-7 of itself
            few = 4 * 2.0 ** -7 * d ** -0.5 * (queries[i].double().abs().amax() * k.abs().amax())
            spread = v.abs().amax(1).repeat_interleave(2, 0)
            assert_within(got, want, bound + 2 * few * spread, f"sequence {s} position {i}")


@pytest.mark.parametrize("capture", [False, True])
def test_serving_a_prompt_and_its_new_tokens(ops, cuda, capture):
    outs, inputs = serve(ops, cuda, 20, capture)
    check_served(outs, inputs, 20)


def test_captured_and_eager_steps_agree_bit_for_bit(ops, cuda):
    for a, b in zip(serve(ops, cuda, 6, False)[0], serve(ops, cuda, 6, True)[0]):
        assert torch.equal(a, b)


def test_two_graphs_and_an_eager_call_at_once(ops, cuda):
    """Captured calls on two streams, replayed at the same time as eager ones on a third: nothing is shared."""
    made = []
    for i, lengths in enumerate(([9000, 20, 4000], [300] * 50, [12000])):
        case = Case(lengths, 2, 128, 64, seed=i, columns=2048)
        query = rows_of((len(lengths), 8, 128), 20 + i, False).to(cuda)
        args = (query, *case.to(cuda), torch.tensor(lengths, device=cuda) - 1)
        made.append((args, ops.paged_decode_attention(*args)))
    graphs = []
    for args, want in made[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.paged_decode_attention(*args)
        graphs.append((graph, out, want, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, out, _, stream in graphs:
            with torch.cuda.stream(stream):
                graph.replay()
        eager = ops.paged_decode_attention(*made[2][0])
        torch.cuda.synchronize()
        assert torch.equal(eager, made[2][1])
        for _, out, want, _ in graphs:
            assert torch.equal(out, want)
            out.zero_()
        torch.cuda.synchronize()


def test_a_workspace_of_the_caller(ops, cuda):
    """Where a call needs one: the queried size is enough, whatever it holds; a smaller one is refused."""
    case = Case([700, 3], 8, 128, 64, columns=2048)
    query = rows_of((2, 16, 128), 1, False).to(cuda)
    keys, values, table = case.to(cuda)
    at = torch.tensor([699, 2], device=cuda)
    want = ops.paged_decode_attention(query, keys, values, table, at)
    need = ops.paged_decode_attention_workspace_bytes(2, 16, 8, 128, 2048 * 64)
    assert need > 0
    held = torch.full((need + 64,), 255, dtype=torch.uint8, device=cuda)
    got = ops.paged_decode_attention(query, keys, values, table, at, workspace=held[:need])
    assert torch.equal(got, want) and held[need:].eq(255).all()
    for bad in (held[:need - 16], held[8:]):
        with pytest.raises(ValueError, match="workspace"):
            ops.paged_decode_attention(query, keys, values, table, at, workspace=bad)
    with pytest.raises(ValueError, match="workspace"):
        ops.paged_decode_attention(query, keys, values, table, at, workspace=held.cpu())


@pytest.mark.parametrize("capacity", [512, 1 << 17], ids=["in-turn", "ranges"])
def test_prompts_repeat_bit_for_bit_captured_and_on_another_stream(ops, cuda, capacity):
    """Eager, replayed and on a second stream at once: the same bits, whichever CTA took which item."""
    counts, starts = [300, 1, 170, 90] * 5, [0, 200, 37, 0] * 5
    made = []
    for seed in range(2):
        case = Case([n + s for n, s in zip(counts, starts)], 8, 128, 64, seed=seed, columns=capacity // 64)
        query = rows_of((sum(counts), 16, 128), 30 + seed, False).to(cuda)
        offsets = torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], device=cuda)
        args = (query, *case.to(cuda), offsets, torch.tensor(starts, device=cuda))
        made.append((args, ops.paged_prefill_attention(*args, out=torch.zeros_like(query))))
    graph, out = torch.cuda.CUDAGraph(), torch.zeros_like(made[0][1])
    with torch.cuda.graph(graph):
        ops.paged_prefill_attention(*made[0][0], out=out)
    side, other = torch.cuda.Stream(), torch.zeros_like(made[1][1])
    torch.cuda.synchronize()
    for _ in range(10):
        out.zero_(), other.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):
            ops.paged_prefill_attention(*made[1][0], out=other)
        torch.cuda.synchronize()
        assert torch.equal(out, made[0][1]) and torch.equal(other, made[1][1])
    assert ops.read_status(cuda) == 0


def test_offsets_past_32_bits(ops, cuda):
    """Pages whose elements lie past 2^31: the write, and both attentions."""
    pages, kv, size, d = 40000, 8, 64, 128          # 2.6e9 elements a pool
    keys, values = (torch.empty(pages, kv, size, d, dtype=BF16, device=cuda) for _ in range(2))
    small = Case([130, 40], kv, d, size, seed=3)
    k, v, table = small.to(cuda)
    high = table.clone()
    for s, n in ((0, 3), (1, 1)):
        for j in range(n):
            high[s, j] = pages - 1 - int(table[s, j])
            keys[high[s, j]], values[high[s, j]] = k[table[s, j]], v[table[s, j]]
    query = rows_of((2, 16, d), 1, False).to(cuda)
    at = torch.tensor([129, 39], device=cuda)
    assert torch.equal(ops.paged_decode_attention(query, keys, values, high, at),
                       ops.paged_decode_attention(query, k, v, table, at))
    prompt = rows_of((170, 16, d), 2, False).to(cuda)
    offsets, starts = torch.tensor([0, 130, 170], device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    assert torch.equal(ops.paged_prefill_attention(prompt, keys, values, high, offsets, starts, out=torch.zeros_like(prompt)),
                       ops.paged_prefill_attention(prompt, k, v, table, offsets, starts, out=torch.zeros_like(prompt)))
    cos, sin = (t.to(cuda) for t in tables(140, d))
    qkv = rows_of((2, 32 * d), 4, False).to(cuda)
    for pool in ((k, v, table), (keys, values, high)):
        ops.paged_qk_norm_rope_kv(qkv, None, None, 1e-6, cos, sin, at, at, pool[2], pool[0], pool[1], q_heads=16,
                                  kv_heads=8, head_dim=d)
    assert torch.equal(keys[high[0, 2], :, 1], k[table[0, 2], :, 1])
    assert torch.equal(values[high[1, 0], :, 39], v[table[1, 0], :, 39])
    assert ops.read_status(cuda) == 0


def test_misaligned_tensors_are_refused(ops, cuda):
    case = Case([20], 2, 64, 16)
    keys, values, table = case.to(cuda)
    odd = torch.zeros(4 * 64 + 1, dtype=BF16, device=cuda)[1:].view(1, 4, 64)
    with pytest.raises(ValueError, match="alignment"):
        ops.paged_decode_attention(odd, keys, values, table, torch.tensor([19], device=cuda))
    out = torch.empty(1, 4, 64, dtype=BF16, device=cuda)
    with pytest.raises(ValueError, match="alignment"):
        ops.paged_prefill_attention(odd, keys, values, table, torch.tensor([0, 1], device=cuda),
                                    torch.tensor([19], device=cuda), out=out)
    strided = torch.zeros(2, 4 * 64 + 4, dtype=BF16, device=cuda)[:, :256].unflatten(1, (4, 64))
    with pytest.raises(ValueError, match="stride"):
        ops.paged_decode_attention(strided, keys, values, table.repeat(2, 1), torch.tensor([19, 19], device=cuda))


def test_an_output_that_is_only_16_byte_aligned(ops, cuda):
    case = Case([150], 2, 64, 16)
    keys, values, table = case.to(cuda)
    query = rows_of((150, 4, 64), 5, False).to(cuda)
    offsets, starts = torch.tensor([0, 150], device=cuda), torch.zeros(1, dtype=torch.int64, device=cuda)
    want = ops.paged_prefill_attention(query, keys, values, table, offsets, starts, out=torch.zeros_like(query))
    out = torch.zeros(150 * 256 + 8, dtype=BF16, device=cuda)[8:].view(150, 4, 64)
    assert torch.equal(ops.paged_prefill_attention(query, keys, values, table, offsets, starts, out=out), want)


def test_prompts_with_odd_offsets_are_flagged(ops, cuda):
    """Row offsets that leave the query or run backwards: that sequence is skipped, the others are right (where a row is
    of two of them, each of its elements is one's or the other's)."""
    case = Case([40, 40, 40], 8, 128, 16)
    query = rows_of((120, 16, 128), 1, False)
    keys, values, table = case.to(cuda)
    starts = torch.zeros(3, dtype=torch.int64, device=cuda)
    for offsets in ([0, 40, 80, 121], [-1, 40, 80, 120], [0, 40, 20, 60]):
        for columns in (3, 3000):
            wide = torch.full((3, columns), -1, dtype=torch.int32, device=cuda)
            wide[:, :3] = table
            out = torch.full_like(query, 5.0, device=cuda)
            ops.paged_prefill_attention(query.to(cuda), keys, values, wide, torch.tensor(offsets, device=cuda), starts,
                                        out=out)
            assert ops.read_status(cuda) == 8
            owners = [s for s in range(3) if 0 <= offsets[s] < offsets[s + 1] <= 120]
            for r in range(120):
                got, near, owned = out[r].double().cpu(), torch.zeros(16, 128, dtype=torch.bool), False
                for s in owners:
                    if offsets[s] <= r < offsets[s + 1]:
                        want, bound = attend(query[r], *case.sequence(s, r - offsets[s] + 1), 128 ** -0.5)
                        near, owned = near | ((got - want).abs() <= bound), True
                assert near.all() if owned else (got == 5).all(), f"{offsets} row {r}"


@pytest.mark.parametrize("count", [400, 1200, 2500])
def test_prompts_that_overlap_are_flagged(ops, cuda, count):
    """Offsets 0, R, 0, R, ...: every other sequence runs backwards, the rest share all rows (and, here, their pages, so
    that a row's result is the same whose ever it is). More tiles than rows in order can have are not looked at."""
    rows = 8192
    case = Case([rows], 1, 64, 64)
    query = rows_of((rows, 1, 64), 1, False)
    keys, values, table = case.to(cuda)
    out = torch.full_like(query, 5.0, device=cuda)
    ops.paged_prefill_attention(query.to(cuda), keys, values, table.repeat(count, 1),
                                torch.tensor([0, rows] * (count // 2) + [0], device=cuda),
                                torch.zeros(count, dtype=torch.int64, device=cuda), out=out)
    assert ops.read_status(cuda) == 8
    for r in [*range(0, rows, 409), rows - 1]:
        want, bound = attend(query[r], *case.sequence(0, r + 1), 0.125)
        assert_within(out[r], want, bound, f"row {r}")


@pytest.mark.parametrize("scale", [0.125, -0.125])
@pytest.mark.parametrize("columns", [3, 3000])
def test_prompts_that_start_far_away(ops, cuda, columns, scale):
    """Starts at the ends of 64 bits: past the table (flagged), or left padding only (zeros)."""
    case = Case([40, 40, 40], 2, 64, 16)
    query = rows_of((120, 4, 64), 1, False)
    keys, values, table = case.to(cuda)
    wide = torch.full((3, columns), -1, dtype=torch.int32, device=cuda)
    wide[:, :3] = table
    offsets = torch.tensor([0, 40, 80, 120], device=cuda)
    for far, status in ((2 ** 63 - 1, 8), (2 ** 63 - 20, 8), (-2 ** 63, 0), (-2 ** 63 + 20, 0)):
        out = torch.full_like(query, 5.0, device=cuda)
        ops.paged_prefill_attention(query.to(cuda), keys, values, wide, offsets, torch.tensor([0, far, 0], device=cuda),
                                    out=out, scale=scale)
        assert ops.read_status(cuda) == status
        if status == 0:
            assert (out[40:80] == 0).all()
        for r in [*range(40), *range(80, 120)]:
            want, bound = attend(query[r], *case.sequence(r // 40, r % 40 + 1), scale)
            assert_within(out[r], want, bound, f"row {r}")


def test_empty_batches_and_given_outputs(ops, cuda):
    case = Case([20], 2, 64, 16)
    keys, values, table = case.to(cuda)
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    query = torch.empty(0, 4, 64, dtype=BF16, device=cuda)
    assert ops.paged_decode_attention(query, keys, values, table[:0], none).shape == (0, 4, 64)
    out = torch.empty_like(query)
    assert ops.paged_prefill_attention(query, keys, values, table[:0], torch.zeros(1, dtype=torch.int64, device=cuda),
                                       none, out=out) is out
    cos, sin = (t.to(cuda) for t in tables(8, 64))
    assert ops.paged_qk_norm_rope_kv(torch.empty(0, 8 * 64, dtype=BF16, device=cuda), None, None, 1e-6, cos, sin, none,
                                     none, table, keys, values, q_heads=4, kv_heads=2, head_dim=64).shape == (0, 4, 64)
    query = rows_of((1, 4, 64), 3, False).to(cuda)
    out = torch.empty_like(query)
    assert ops.paged_decode_attention(query, keys, values, table, torch.tensor([19], device=cuda), out=out) is out
    assert_within(out[0], *attend(query[0].cpu(), *case.sequence(0, 20), 0.125))
