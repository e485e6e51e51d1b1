"""A PagedCache holds its tensors' addresses: given other memory they are refused, before a kernel reads the old."""

import pytest

torch = pytest.importorskip("torch")


def _moves(t):
    t.data = torch.zeros_like(t)


def _sets(t):
    t.set_(torch.ones_like(t))


def _frees(t):
    t.untyped_storage().resize_(0)


@pytest.mark.parametrize("move", [_moves, _sets, _frees])
@pytest.mark.parametrize("bits,name", [(16, "k"), (16, "v"), (4, "k"), (4, "v"), (4, "k_scale"), (4, "v_scale")])
def test_a_cache_whose_tensors_moved_is_refused(move, bits, name):
    from pdum_dsl_amd import kernels as K

    cache = K.paged_cache(3, 2, 16, 64, bits=bits, device="cpu")
    i32 = torch.int32
    t = (torch.zeros((1, 3), dtype=i32), torch.zeros(2, dtype=i32), torch.zeros(1, dtype=i32))
    x = torch.zeros((1, 2, 64), dtype=torch.bfloat16)
    calls = (lambda: K.paged_append(x, x, cache, *t), lambda: K.paged_rows(cache, *t, 1), lambda: K.paged_attention(x, cache, *t))
    for call in calls:
        with pytest.raises(ValueError, match="CPU tensor"):  # as far as a call gets here
            call()
    getattr(cache, name).add_(1)  # its contents are the calls'
    for call in calls:
        with pytest.raises(ValueError, match="CPU tensor"):
            call()
    move(getattr(cache, name))
    for call in calls:
        with pytest.raises(ValueError, match="moved"):
            call()
    again = K.PagedCache(*(None if p is None else p.clone() if p.untyped_storage().nbytes() else torch.zeros(p.shape, dtype=p.dtype)
                           for p in (cache.k, cache.v, cache.k_scale, cache.v_scale)), cache.dtype)
    with pytest.raises(ValueError, match="CPU tensor"):
        K.paged_attention(x, again, *t)
