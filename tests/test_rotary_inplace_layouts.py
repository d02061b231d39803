"""Which q and k rotary turns in place: those that share no element, wherever they lie
in one tensor."""
import itertools

import pytest
import torch


def _elements(t):
    at = torch.zeros(t.shape, dtype=torch.int64) + t.storage_offset()
    for i, (n, s) in enumerate(zip(t.shape, t.stride())):
        at += (torch.arange(n) * s).view([-1 if j == i else 1 for j in range(t.dim())])
    return set(at.flatten().tolist())


def _parts(b, n, first, second, d, layout):
    """Two parts of a tensor with heads between tokens and values."""
    heads = first + second + 1
    if layout == "tokens":
        t = torch.zeros(b, n, heads, d)
        return t[:, :, :first], t[:, :, first:first + second]
    if layout == "heads":
        t = torch.zeros(b, heads, n, d).transpose(1, 2)
        return t[:, :, :first], t[:, :, first:first + second]
    t = torch.zeros(b, n, heads * d)
    return t[..., :first * d].view(b, n, first, d), t[..., first * d:(first + second) * d].view(b, n, second, d)


@pytest.mark.parametrize("layout", ["tokens", "heads", "flat"])
@pytest.mark.parametrize("b,n", [(1, 1), (1, 5), (3, 1), (2, 4)])
@pytest.mark.parametrize("first,second", [(4, 4), (4, 1), (1, 4), (2, 3), (3, 2), (1, 1)])
def test_parts_of_one_tensor_are_apart(first, second, b, n, layout):
    from quant_models import ops

    x, y = _parts(b, n, first, second, 6, layout)
    assert not _elements(x) & _elements(y)
    assert ops._apart_from(x, y) and ops._apart_from(y, x)


def test_what_is_called_apart_shares_nothing():
    """Every pair of views of a small tensor: never apart where an element is shared."""
    from quant_models import ops

    base, views = torch.zeros(72), []
    for shape, strides in (((2, 3, 2, 2), (24, 8, 4, 1)), ((2, 3, 1, 2), (24, 8, 4, 1)), ((2, 3, 2, 2), (24, 8, 2, 1)), ((1, 3, 2, 2), (1, 8, 4, 1)),
                           ((2, 1, 3, 2), (12, 5, 4, 1)), ((2, 3, 2, 2), (4, 8, 2, 1)), ((2, 2, 2, 2), (16, 4, 8, 1)), ((1, 1, 1, 2), (3, 7, 9, 1))):
        reach = sum((n - 1) * s for n, s in zip(shape, strides))
        views += [base.as_strided(shape, strides, at) for at in range(0, 72 - reach, 1)][:26]
    apart = 0
    for x, y in itertools.combinations(views, 2):
        if ops._apart_from(x, y):
            apart += 1
            assert not _elements(x) & _elements(y), (x.shape, x.stride(), x.storage_offset(), y.shape, y.stride(), y.storage_offset())
    assert apart > 1000


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["q first", "k first"])
def test_grouped_heads_turn_where_they_lie(order):
    """q and fewer k heads in one tensor, in either order."""
    from quant_models import ops

    qkv = torch.randn(2, 7, 4 + 1 + 1, 32, device="cuda").half()
    q, k = (qkv[:, :, :4], qkv[:, :, 4:5]) if order == "q first" else (qkv[:, :, 1:5], qkv[:, :, :1])
    positions, freqs = torch.arange(7, device="cuda"), ops.rotary_frequencies((16,))
    want, rest = ops.rotary((q.clone(), k.clone()), positions, freqs), qkv[:, :, 5].clone()
    ops.rotary((q, k), positions, freqs, inplace=True)
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, :, 5], rest)
