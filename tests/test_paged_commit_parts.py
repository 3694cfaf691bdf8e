"""A commit over more caches than one launch takes (a model of many layers) is one call:
what it refuses, it refuses before any layer is moved."""
import pytest
import torch

from nanokv_amd import _lib, ops

LAYERS = _lib.NKV_PAGED_CACHES + 2


@pytest.fixture
def launches(monkeypatch):
    """The C calls that would be made (device checks aside, which need a GPU)."""
    made = []
    monkeypatch.setattr(ops, "_require_gpu", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(ops, "_device_call", lambda name, device, *a: made.append(a[0]._obj.n_caches))
    return made


def layers(n=LAYERS):
    return [ops.PagedCache.empty(2, 16, 1, 8, torch.device("cpu")) for _ in range(n)]


def commit(caches, **kw):
    i32 = torch.int32
    return ops.paged_commit(**{**dict(caches=caches, table=torch.zeros((2, 4), dtype=i32), start=0,
                                      rows=torch.zeros((2, 3), dtype=i32)), **kw})


def storage(numel):
    """bf16 elements from a 16-byte boundary on."""
    x = torch.zeros(numel + 8, dtype=torch.bfloat16)
    at = -x.data_ptr() % 16 // 2
    return x[at:at + numel]


def pool_at(x, offset):
    return x[offset:offset + 256].view(2, 1, 16, 8)


def test_many_layers_are_launched_in_parts(launches):
    assert commit(layers()).shape == (2,)
    assert launches == [_lib.NKV_PAGED_CACHES, 2]


@pytest.mark.parametrize("later", [_lib.NKV_PAGED_CACHES, LAYERS - 1])
@pytest.mark.parametrize("earlier", [0, 1, _lib.NKV_PAGED_CACHES - 1])
def test_a_layer_named_twice_is_refused(launches, earlier, later):
    caches = layers()
    caches[later] = caches[earlier]
    with pytest.raises(ValueError, match="overlap"):
        commit(caches)
    caches[later] = ops.PagedCache(layers(1)[0].k, caches[earlier].k)
    with pytest.raises(ValueError, match="overlap"):
        commit(caches)
    assert not launches


def test_layers_that_share_a_part_of_their_memory_are_refused(launches):
    x = storage(1024)
    caches = layers()
    caches[3].k = pool_at(x, 0)
    caches[-1].v = pool_at(x, 248)
    with pytest.raises(ValueError, match="overlap"):
        commit(caches)
    assert not launches
    caches[-1].v = pool_at(x, 256)            # the next to it
    commit(caches)
    assert len(launches) == 2


def test_a_later_layer_that_is_not_aligned_is_refused(launches):
    caches = layers()
    caches[-1].k = pool_at(storage(1024), 4)
    with pytest.raises(ValueError, match="aligned"):
        commit(caches)
    assert not launches


@pytest.mark.parametrize("name", ["table", "rows", "start", "counts"])
def test_a_later_layer_over_what_the_call_reads_is_refused(launches, name):
    x = storage(1024)
    caches = layers()
    caches[-1].v = pool_at(x, 0)
    words = x.view(torch.int32)
    shape = {"table": (2, 4), "rows": (2, 3)}.get(name, (2,))
    n = shape[0] * (shape[1] if len(shape) == 2 else 1)
    inside = {name: words[127:127 + n].view(shape)}
    with pytest.raises(ValueError, match="overlap"):
        commit(caches, **inside)
    assert not launches
    commit(caches, **{name: words[128:128 + n].view(shape)})    # behind it
    assert len(launches) == 2


def test_nothing_to_be_moved(launches):
    caches = layers()
    caches[-1] = caches[0]
    empty = torch.zeros((0, 4), dtype=torch.int32)
    assert commit(caches, table=empty, rows=empty[:, :3]).shape == (0,)


@pytest.mark.gpu
def test_a_refused_commit_moves_nothing(dev):
    g = torch.Generator().manual_seed(3)
    caches = [ops.PagedCache(*(torch.randn((2, 1, 16, 8), generator=g).to(torch.bfloat16).to(dev)
                               for _ in range(2))) for _ in range(LAYERS)]
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=dev)
    rows = torch.tensor([[4, 2, 0]], dtype=torch.int32, device=dev)
    before = [(c.k.clone(), c.v.clone()) for c in caches]
    with pytest.raises(ValueError, match="overlap"):
        ops.paged_commit(caches[:-1] + caches[:1], table, 14, rows)
    for c, (k, v) in zip(caches, before):
        assert torch.equal(c.k, k) and torch.equal(c.v, v)
    assert ops.paged_commit(caches, table, 14, rows).tolist() == [17]
    for c, pools in zip(caches, before):
        for new, old in zip((c.k, c.v), pools):
            old[1, 0, 14:16], old[0, 0, 0] = old[0, 0, [2, 0]].clone(), old[1, 0, 14].clone()
            assert torch.equal(new, old)
