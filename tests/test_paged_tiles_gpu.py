"""The tiled form of the paged prompt attention: what the cases of the row form do not reach."""
import pytest
import torch

from tests.paged_reference import BF16, Case, assert_within, attend, rng

pytestmark = pytest.mark.gpu

# Table widths with which prompts of hundreds of rows go in whole items, and in even ranges of key tiles
WIDTHS = pytest.mark.parametrize("capacity", [None, 1 << 17], ids=["in-turn", "ranges"])
HEADS = pytest.mark.parametrize("q,kv,d", [(16, 8, 128), (16, 8, 64), (12, 4, 64)])


@pytest.fixture(scope="module")
def ops(cuda):
    from qwen3_tts_b200 import ops as _ops
    return _ops


def prompt(ops, cuda, case, query, rows, start=0, out=None):
    """One sequence's `rows` rows from position `start` on; the status has to stay clear."""
    keys, values, table = case.to(cuda)
    out = torch.empty_like(query, device=cuda) if out is None else out
    ops.paged_prefill_attention(query.to(cuda), keys, values, table, torch.tensor([0, rows], device=cuda),
                                torch.tensor([start], device=cuda), out=out)
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
        got = prompt(ops, cuda, case, query, rows)
        keys, values = case.sequence(0, rows)
        for r in {0, where - 1, where, where + 1, *range(where % 64, rows, 64), rows - 1}:
            if r >= where and score != -float("inf"):
                assert got[r].isnan().all(), f"key {where} row {r}"
                continue
            seen = [j for j in range(r + 1) if j != where]
            want, bound = attend(query[r], keys[:, seen], values[:, seen], d ** -0.5)
            assert_within(got[r], want, bound, f"key {where} row {r}")


def test_every_item_is_taken_over_once(ops, cuda):
    """Thousands of items of a few rows: a CTA takes over a hundred, one answer after the other in the same place."""
    counts = [1 + i % 4 for i in range(2000)]
    case = Case([8] * 16, 8, 128, 16)
    keys, values, table = case.to(cuda)
    rows = sum(counts)
    query = torch.randn(rows, 16, 128, generator=rng(5)).to(BF16)
    offsets = torch.tensor([0, *counts]).cumsum(0)
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
    got = ops.paged_prefill_attention(query, keys, values, table[kind], offsets, torch.tensor(starts, device=cuda)[kind],
                                      out=torch.full_like(query, float("nan")))
    assert ops.read_status(cuda) == 0
    for r in range(0, rows, 1 << 19):
        part, index = got[r:r + (1 << 19)], row[r:r + (1 << 19)]
        assert ((part.double() - want[index]).abs() <= bound[index]).all(), f"rows from {r} on"
