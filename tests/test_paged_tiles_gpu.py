"""The tiled form of the paged prompt attention: what the cases of the row form do not reach."""
import pytest
import torch

from tests.paged_reference import BF16, Case, assert_within, attend, rng
from tests.test_paged_gpu import check_prompt

pytestmark = pytest.mark.gpu

# Table widths with which prompts of hundreds of rows go in whole items, and in even ranges of key tiles
WIDTHS = pytest.mark.parametrize("capacity", [None, 1 << 17], ids=["in-turn", "ranges"])
HEADS = pytest.mark.parametrize("q,kv,d", [(16, 8, 128), (16, 8, 64), (12, 4, 64)])


@pytest.fixture(scope="module")
def ops(cuda):
    from qwen3_tts_b200 import ops as _ops
    return _ops


def form_of(ops, query, case, sequences=1):
    return ops.paged_prefill_attention_form(*query.shape[:1], sequences, query.shape[1], case.kv_heads, case.dim,
                                            case.table.shape[1] * case.page)


def form_for(capacity):
    return "tiles" if capacity is None else "ranges"


def prompt(ops, cuda, case, query, form):
    """One sequence from position 0 on, in the form that the test is meant for; the status has to stay clear."""
    assert form_of(ops, query, case) == form
    keys, values, table = case.to(cuda)
    out = torch.full_like(query, float("nan"), device=cuda)
    ops.paged_prefill_attention(query.to(cuda), keys, values, table, torch.tensor([0, len(query)], device=cuda),
                                torch.tensor([0], device=cuda), out=out)
    assert ops.read_status(cuda) == 0
    return out.cpu()


def case_of(length, kv, d, page, capacity, seed):
    return Case([length], kv, d, page, seed=seed, columns=None if capacity is None else capacity // page)


@WIDTHS
@HEADS
@pytest.mark.parametrize("score", [float("nan"), float("inf"), -float("inf")])
def test_scores_that_are_not_finite_follow_the_formula(ops, cuda, q, kv, d, capacity, score):
    """One key whose scores are NaN or +inf leaves no value to the rows that see it, wherever it stands, and does not
    touch the others; one of -inf has weight 0."""
    rows = 700
    query = torch.randn(rows, q, d, generator=rng(3)).to(BF16)
    query[..., 0] = query[..., 0].abs() + 0.25
    for where in (1, 6, 7, 23, 64, 102, 103, 135, 383, 620):
        case = case_of(rows, kv, d, 16, capacity, where)
        case.keys[case.table[0, where // 16], :, where % 16, 0] = score
        got = prompt(ops, cuda, case, query, form_for(capacity))
        keys, values = case.sequence(0, rows)
        for r in {0, where - 1, where, where + 1, *range(where % 64, rows, 64), rows - 1}:
            if r >= where and score != -float("inf"):
                assert got[r].isnan().all(), f"key {where} row {r}"
                continue
            seen = [j for j in range(r + 1) if j != where]
            want, bound = attend(query[r], keys[:, seen], values[:, seen], d ** -0.5)
            assert_within(got[r], want, bound, f"key {where} row {r}")


@pytest.mark.parametrize("q,kv,d", [(16, 8, 128), (16, 1, 64), (9, 1, 64)])
@pytest.mark.parametrize("columns", [4, 60])
@pytest.mark.parametrize("score", [float("nan"), float("inf"), -float("inf")])
def test_scores_that_are_not_finite_by_rows(ops, cuda, q, kv, d, columns, score):
    """The same where few rows go by rows, each alone or several in a pass over the keys."""
    rows = 45
    query = torch.randn(rows, q, d, generator=rng(3)).to(BF16)
    query[..., 0] = query[..., 0].abs() + 0.25
    for where in (1, 6, 16, 31, 40):
        case = Case([rows], kv, d, 16, seed=where, columns=columns)
        case.keys[case.table[0, where // 16], :, where % 16, 0] = score
        got = prompt(ops, cuda, case, query, "rows")
        keys, values = case.sequence(0, rows)
        for r in range(rows):
            if r >= where and score != -float("inf"):
                assert got[r].isnan().all(), f"key {where} row {r}"
                continue
            seen = [j for j in range(r + 1) if j != where]
            assert_within(got[r], *attend(query[r], keys[:, seen], values[:, seen], d ** -0.5), f"key {where} row {r}")


def test_every_item_is_taken_over_once(ops, cuda):
    """Thousands of items of a few rows: a CTA takes over a hundred, one answer after the other in the same place."""
    counts = [1 + i % 4 for i in range(2000)]
    case = Case([8] * 16, 8, 128, 16)
    keys, values, table = case.to(cuda)
    rows = sum(counts)
    query = torch.randn(rows, 16, 128, generator=rng(5)).to(BF16)
    offsets = torch.tensor([0, *counts]).cumsum(0)
    assert form_of(ops, query, case, 2000) == "tiles"
    args = (query.to(cuda), keys, values, table.repeat(125, 1), offsets.to(cuda),
            torch.tensor([i % 5 for i in range(2000)], device=cuda))
    want = ops.paged_prefill_attention(*args, out=torch.full_like(args[0], float("nan")))
    for _ in range(20):
        assert torch.equal(ops.paged_prefill_attention(*args, out=torch.full_like(args[0], float("nan"))), want)
    assert ops.read_status(cuda) == 0 and want.isfinite().all()
    for s in range(0, 2000, 7):
        r = int(offsets[s + 1]) - 1
        keys, values = case.sequence(s % 16, s % 5 + counts[s])
        assert_within(want[r], *attend(query[r], keys, values, 128 ** -0.5), f"sequence {s}")


@pytest.mark.parametrize("count,period", [(2100, 301), (4097, 301), (50001, 331), (1 << 20, 48)])
def test_sequences_by_the_thousand(ops, cuda, count, period):
    """Sequence s is as s % period (its pages, length, start and queries), so that all rows are known from a few: up to
    5 rows, one of the period none and one, where there are few sequences, several query tiles."""
    counts = [(7 * i) % 6 for i in range(period)]
    if count < 10000:
        counts[period // 2] = 300
    starts, lengths = [(5 * i) % 40 for i in range(period)], [n + 40 for n in counts]
    case = Case(lengths, 1, 64, 16, seed=period)
    first = torch.tensor([0, *counts]).cumsum(0)
    small = torch.randn(int(first[-1]), 2, 64, generator=rng(period + 1)).to(BF16)
    known = [attend(small[int(first[s]) + i], *case.sequence(s, starts[s] + i + 1), 0.125)
             for s in range(period) for i in range(counts[s])]
    want, bound = (torch.stack(x).to(cuda) for x in zip(*known))
    kind = torch.arange(count, device=cuda) % period
    many = torch.tensor(counts, device=cuda)[kind]
    offsets = torch.cat((many.new_zeros(1), many.cumsum(0)))
    rows = int(offsets[-1])
    sequence = torch.repeat_interleave(torch.arange(count, device=cuda), many)
    row = first.to(cuda)[kind[sequence]] + torch.arange(rows, device=cuda) - offsets[sequence]
    keys, values, table = case.to(cuda)
    query = small.to(cuda)[row]
    assert form_of(ops, query, case, count) == "tiles"
    got = ops.paged_prefill_attention(query, keys, values, table[kind], offsets, torch.tensor(starts, device=cuda)[kind],
                                      out=torch.full_like(query, float("nan")))
    assert ops.read_status(cuda) == 0
    for r in range(0, rows, 1 << 19):
        part, index = got[r:r + (1 << 19)], row[r:r + (1 << 19)]
        assert ((part.double() - want[index]).abs() <= bound[index]).all(), f"rows from {r} on"


@WIDTHS
@HEADS
def test_rising_scores_rescale_the_output(ops, cuda, q, kv, d, capacity):
    """Maxima that pass the lazy margin (8 powers of two) by a little and by much from key tile to key tile, up and down,
    each row's at tiles of its own. Where a single key passes it by a little, the 128 keys of the tile before keep a
    third of the weight, and values around 1 show a wrong factor of the output as well as of the sum."""
    rows = 900
    case = case_of(rows, kv, d, 32, capacity, 1)
    level = torch.full((rows,), -30.0)
    for tile, (all_keys, one) in enumerate([(0, None), (None, 5.8), (5.0, None), (None, 11.6), (-4, 9.0), (30, None), (10, 33)]):
        if all_keys is not None:
            level[128 * tile:128 * (tile + 1)] = all_keys
        if one is not None:
            level[128 * tile + 17 * tile % 128] = one
    at = torch.arange(rows)
    noise = 0.02 * torch.randn(rows, kv, d, generator=rng(2))
    case.keys[case.table[0, at // 32].long(), :, at % 32] = (level[:, None, None] * d ** -0.5 + noise).to(BF16)
    case.values += 1
    slope = torch.tensor([1.0, 1.0, 0.96, 1.05, -1.0, 0.5, 1.5, 0.0])[at * 7 // 5 % 8]
    query = (slope[:, None, None] + 0.02 * torch.randn(rows, q, d, generator=rng(4))).to(BF16)
    got = prompt(ops, cuda, case, query, form_for(capacity))
    keys, values = case.sequence(0, rows)
    for r in range(0, rows, 3):
        assert_within(got[r], *attend(query[r], keys[:, :r + 1], values[:, :r + 1], d ** -0.5), f"row {r}")


@WIDTHS
@HEADS
@pytest.mark.parametrize("scale", [0.5, 1e-3, 1e-30])
def test_scales_in_tiles(ops, cuda, q, kv, d, capacity, scale):
    columns = 45 if capacity is None else capacity // 16
    assert ops.paged_prefill_attention_form(703, 1, q, kv, d, columns * 16) == form_for(capacity)
    check_prompt(ops, cuda, q, kv, d, 16, [700], [0], scale=scale, columns=columns, lead=1, tail=2)


@WIDTHS
@pytest.mark.parametrize("d", [64, 128])
def test_bad_pages_in_tiles_are_flagged(ops, cuda, d, capacity):
    """The rows that need the page are unspecified; their neighbours are right and nothing faults."""
    lengths = [300, 300, 300]
    case = Case(lengths, 8, d, 16, columns=None if capacity is None else capacity // 16)
    query = torch.randn(900, 16, d, generator=rng(1)).to(BF16)
    assert form_of(ops, query, case, 3) == form_for(capacity)
    keys, values, table = case.to(cuda)
    offsets, zero = torch.tensor([0, 300, 600, 900], device=cuda), torch.zeros(3, dtype=torch.int64, device=cuda)

    def run(page_table, start=zero):
        got = ops.paged_prefill_attention(query.to(cuda), keys, values, page_table, offsets, start,
                                          out=torch.zeros_like(query, device=cuda))
        for r in [*range(0, 300, 7), 299, *range(600, 900, 7), 899]:
            want, bound = attend(query[r], *case.sequence(r // 300, r % 300 + 1), d ** -0.5)
            assert_within(got[r], want, bound, f"row {r}")
        return ops.read_status(cuda), got

    assert run(table)[0] == 0
    for column, entry in ((1, len(case.keys)), (9, -1), (18, (1 << 31) - 1), (0, -(1 << 31))):
        bad = table.clone()
        bad[1, column] = entry
        status, got = run(bad)
        assert status == 8
        for r in range(300, 300 + 16 * column - 127, 31):  # key tiles before the page's: not touched either
            assert_within(got[r], *attend(query[r], *case.sequence(1, r - 299), d ** -0.5), f"row {r}")
    past = torch.tensor([0, table.shape[1] * 16 - 150, 0], device=cuda)   # the second half of the rows past the table
    assert run(table, past)[0] == 8


@WIDTHS
def test_offsets_and_starts_that_make_no_sense_in_tiles(ops, cuda, capacity):
    """A sequence whose offsets leave the query or run backwards is skipped, a start at the ends of 64 bits is past the
    table (flagged) or padding (zeros); the other sequences are right."""
    case = Case([300, 300, 300], 8, 128, 16, columns=None if capacity is None else capacity // 16)
    query = torch.randn(900, 16, 128, generator=rng(1)).to(BF16)
    assert form_of(ops, query, case, 3) == form_for(capacity)
    keys, values, table = case.to(cuda)

    def run(offsets, starts, sequences, shared=()):
        out = torch.full_like(query, 5.0, device=cuda)
        ops.paged_prefill_attention(query.to(cuda), keys, values, table, torch.tensor(offsets, device=cuda),
                                    torch.tensor(starts, device=cuda), out=out)
        for s in sequences:
            for i in [*range(0, offsets[s + 1] - offsets[s], 11), offsets[s + 1] - offsets[s] - 1]:
                r = offsets[s] + i
                if r not in shared:
                    assert_within(out[r], *attend(query[r], *case.sequence(s, i + 1), 128 ** -0.5), f"row {r}")
        return ops.read_status(cuda), out

    status, out = run([0, 300, 600, 901], [0, 0, 0], (0, 1))
    assert status == 8 and (out[600:] == 5).all()
    status, out = run([-1, 300, 600, 900], [0, 0, 0], (1, 2))
    assert status == 8 and (out[:300] == 5).all()
    status, out = run([0, 300, 290, 590], [0, 0, 0], (0, 2), shared=range(290, 300))
    assert status == 8 and (out[590:] == 5).all()
    for r in range(290, 300):   # rows of two sequences: each element is one's or the other's
        near = [(out[r].double().cpu() - want).abs() <= bound for want, bound in
                (attend(query[r], *case.sequence(s, r - first + 1), 128 ** -0.5) for s, first in ((0, 0), (2, 290)))]
        assert (near[0] | near[1]).all(), f"row {r}"
    status, out = run([0, 2 ** 62, 600, 900], [0, 0, 0], (2,))
    assert status == 8 and (out[:600] == 5).all()
    for far, flag in ((2 ** 63 - 1, 8), (2 ** 63 - 200, 8), (2 ** 31, 8), (-2 ** 63, 0), (-2 ** 31 - 7, 0), (-300, 0)):
        status, out = run([0, 300, 600, 900], [0, far, 0], (0, 2))
        assert status == flag and (flag or (out[300:600] == 0).all())


@WIDTHS
@pytest.mark.parametrize("d", [64, 128])
def test_an_output_in_tiles_that_is_only_16_byte_aligned(ops, cuda, d, capacity):
    case = Case([700], 8, d, 16, columns=None if capacity is None else capacity // 16)
    query = torch.randn(700, 16, d, generator=rng(5)).to(BF16)
    want = prompt(ops, cuda, case, query, form_for(capacity))
    keys, values, table = case.to(cuda)
    whole = torch.full((700 * 16 * d + 16,), 5.0, dtype=BF16, device=cuda)
    out = whole[8:-8].view(700, 16, d)
    assert out.data_ptr() % 32 == 16
    ops.paged_prefill_attention(query.to(cuda), keys, values, table, torch.tensor([0, 700], device=cuda),
                                torch.tensor([0], device=cuda), out=out)
    assert torch.equal(out.cpu(), want) and (whole[:8] == 5).all() and (whole[-8:] == 5).all()


@WIDTHS
def test_offsets_past_32_bits_in_tiles(ops, cuda, capacity):
    """Pages whose elements lie past 2^31 and 2^32."""
    pages, kv, size, d = 70000, 8, 64, 128          # 4.6e9 elements a pool
    keys, values = (torch.empty(pages, kv, size, d, dtype=BF16, device=cuda) for _ in range(2))
    case = Case([500, 300], kv, d, size, seed=3, columns=None if capacity is None else capacity // size)
    k, v, table = case.to(cuda)
    high = table.clone()
    for s, n in enumerate(case.lengths):
        for j in range(-(-n // size)):
            high[s, j] = pages - 1 - 2000 * int(table[s, j])
            keys[high[s, j]], values[high[s, j]] = k[table[s, j]], v[table[s, j]]
    query = torch.randn(800, 16, d, generator=rng(2)).to(BF16)
    assert form_of(ops, query, case, 2) == form_for(capacity)
    rest = torch.tensor([0, 500, 800], device=cuda), torch.zeros(2, dtype=torch.int64, device=cuda)
    query = query.to(cuda)
    assert torch.equal(ops.paged_prefill_attention(query, keys, values, high, *rest, out=torch.zeros_like(query)),
                       ops.paged_prefill_attention(query, k, v, table, *rest, out=torch.zeros_like(query)))
    assert ops.read_status(cuda) == 0


@pytest.mark.parametrize("rows,capacity", [(1, 8 * 6144), (3, 8 * 6144), (9, 4 * 6144), (18, 2 * 6144), (60, 6144), (100, 2048)])
def test_prompts_on_both_sides_of_the_limit_for_rows(ops, cuda, rows, capacity):
    """16 query and 8 KV heads: by rows up to 6144 keys of the table for each CTA that shares an item, up to 2048 where
    items are more than SMs, in tiles past them. The same results."""
    for columns, by_rows in ((capacity // 64, True), (capacity // 64 + 1, False)):
        assert (ops.paged_prefill_attention_form(rows, 1, 16, 8, 128, 64 * columns) == "rows") == by_rows
        check_prompt(ops, cuda, 16, 8, 128, 64, [rows], [1500], columns=columns)


def test_prompts_on_both_sides_of_the_limit_for_items(ops, cuda):
    """By rows up to three items (4 rows of one of 8 KV heads) an SM of 148."""
    for rows, by_rows in ((216, True), (220, False)):
        assert (ops.paged_prefill_attention_form(rows, 1, 16, 8, 128, 2048) == "rows") == by_rows
        check_prompt(ops, cuda, 16, 8, 128, 64, [rows], [1800], columns=32)


@WIDTHS
@HEADS
def test_queries_that_are_not_finite_stay_in_their_rows(ops, cuda, q, kv, d, capacity):
    """NaN and infinite queries, of a sequence or of nobody, in the tiles of others."""
    case = Case([500, 400], kv, d, 16, columns=None if capacity is None else capacity // 16)
    query = torch.randn(930, q, d, generator=rng(8)).to(BF16)
    bad = [70, 71, 199, 444]
    query[:10] = query[510:520] = query[920:] = float("nan")
    for r, value in zip(bad, (float("nan"), float("inf"), -float("inf"), float("nan"))):
        query[r, :, 3] = value
    assert form_of(ops, query, case, 4) == form_for(capacity)
    keys, values, table = case.to(cuda)
    out = torch.full_like(query, 5.0, device=cuda)
    ops.paged_prefill_attention(query.to(cuda), keys, values, table[[0, 0, 1, 1]].contiguous(),
                                torch.tensor([10, 510, 520, 920, 920], device=cuda), torch.tensor([0, 0, 0, 0], device=cuda),
                                out=out)
    # rows 510 .. 519 belong to sequence 1 of four: finite keys, queries that are not
    assert ops.read_status(cuda) == 0 and out[510:520].isnan().all()
    assert (out[:10] == 5).all() and (out[920:] == 5).all()
    for s, first, n in ((0, 10, 500), (1, 520, 400)):
        for i in range(n):
            if first + i in bad:
                # a dim of +-inf scores +-inf by the key's sign: with both signs seen, some score is +inf
                assert out[first + i].isnan().all()
            elif i % 7 == 0 or first + i + 1 in bad or first + i - 1 in bad:
                assert_within(out[first + i], *attend(query[first + i], *case.sequence(s, i + 1), d ** -0.5), f"row {first + i}")
