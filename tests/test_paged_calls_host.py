"""Calls of the paged cache operators that are allowed although their tensors look unusual, and the refusal of those that
are not, up to the launch (no GPU)."""
import pytest
import torch

from qwen3_tts_b200 import _lib, ops
from tests.test_paged_host import BF16, FakeCuda, decode, index, no_launch, pool, prompt, table, write  # noqa: F401


def odd(t, dim):
    """t with a stride of 8 in a dim of one element, where no stride matters."""
    assert t.shape[dim] == 1
    stride = list(t.stride())
    stride[dim] = 8
    return torch.as_strided(t, t.shape, stride)


def zeros(*shape):
    return torch.zeros(*shape, dtype=BF16)


ONE_ROW = dict(query=odd(zeros(1, 4, 64), 0), positions=index(1), out=zeros(1, 4, 64))
ONE_HEAD = dict(keys=odd(pool(heads=1), 1), values=pool(heads=1))
ONE_PAGE = dict(keys=pool(pages=1), values=odd(pool(pages=1), 0))


@pytest.mark.parametrize("entry,change", [
    (decode, ONE_ROW), (decode, ONE_ROW | dict(page_table=odd(table(rows=1), 0))), (decode, ONE_HEAD), (decode, ONE_PAGE),
    (decode, dict(page_table=odd(table(columns=1), 1))),
    (decode, dict(query=odd(zeros(3, 1, 64), 1), out=zeros(3, 1, 64), **ONE_HEAD)),
    (prompt, dict(query=odd(zeros(1, 4, 64), 0), out=zeros(1, 4, 64))), (prompt, ONE_HEAD), (prompt, ONE_PAGE),
    (write, dict(qkv=odd(zeros(1, 512), 0), rotary=index(1), at=index(1), sequences=None, out=zeros(1, 4, 64))),
    (write, ONE_PAGE)])
def test_a_dim_of_one_element_has_any_stride(entry, change, no_launch, monkeypatch):  # noqa: F811
    """The call gets the strides of a dense layout for it."""
    def call(name, packed, device):
        layout = {decode: _lib.PAGED_DECODE, prompt: _lib.PAGED_PREFILL, write: _lib.PAGED_WRITE}[entry]
        raise no_launch(layout.unpack(packed))

    monkeypatch.setattr(ops, "_paged_call", call)
    with pytest.raises(no_launch) as reached:
        entry(**change)
    fields = reached.value.args[0]
    page_stride, pages, size, heads, dim, _, table_stride, table_rows, columns = fields[2:11]
    assert page_stride == heads * size * dim and (table_rows == 1 or table_stride == columns)
    rows, q_heads = fields[14:16]
    assert fields[13] == (q_heads + (2 * heads if entry is write else 0)) * dim


def test_a_prompt_needs_an_output():
    pages = [FakeCuda(pool()), FakeCuda(pool())]
    with pytest.raises(ValueError, match="out must be given"):
        ops.paged_prefill_attention(FakeCuda(zeros(9, 4, 64)), *pages, FakeCuda(table()), FakeCuda(index(4)),
                                    FakeCuda(index(3)), out=None)


def test_the_form_of_a_prompt():
    form = ops.paged_prefill_attention_form
    assert form(13, 1, 8, 8, 64, 16) == "rows" and form(8191, 1, 32, 8, 128, 8192) == "tiles"
    assert form(700, 1, 16, 8, 128, 1 << 17) == "ranges"
    assert form(8191, 1, 32, 8, 128, (1 << 26) + 16) == "rows"     # more keys than the tiles count
    for bad in ((0, 1, 8, 8, 64, 16), (13, 0, 8, 8, 64, 16), (13, 1, 4, 8, 64, 16), (13, 1, 8, 0, 64, 16), (13, 1, 8, 8, 64, 0)):
        with pytest.raises(ValueError, match="geometry"):
            form(*bad)
