"""What the paged-cache calls refuse, on the CPU: every check comes before any device work."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
from sensenova_b200 import ffi, paged  # noqa: E402
from sensenova_b200.ffi import SnlError  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def make(d=256, page=16, kv=2, heads=8, rows=3, dtype=F16, pages=4, weight=True):
    k, v = (torch.zeros(pages, kv, page, d, dtype=dtype) for _ in range(2))
    w = torch.zeros(pages, kv, page) if weight else None
    table = torch.zeros(1, 4, dtype=torch.int32)
    batch = paged.PagedBatch(table, torch.tensor([0, rows], dtype=torch.int32), torch.tensor([9], dtype=torch.int32),
                             rows, 9)
    q = torch.zeros(rows, heads, d, dtype=dtype)
    return paged.PagedCache(k, v, w), batch, q


def attend(cache, batch, q, out=None, work=None, **kw):
    out = torch.zeros_like(q) if out is None else out
    n = cache.attend_workspace(batch, q.shape[1]) if work is None else work
    cache.attend(batch, q, out, torch.zeros(max(n, 0), dtype=torch.uint8), **kw)


def refused(kind, match, call, *a, **kw):
    with pytest.raises(SnlError, match=match) as e:
        call(*a, **kw)
    assert e.value.kind == kind


@pytest.mark.parametrize("kw,kind,match", [
    (dict(d=64), "SNL_E_UNSUPPORTED", "head_dim must be 128 or 256"),
    (dict(page=4), "SNL_E_UNSUPPORTED", "page_size must be a power of two of at least 8"),
    (dict(page=24), "SNL_E_UNSUPPORTED", "page_size must be a power of two of at least 8"),
    (dict(dtype=F32), "SNL_E_UNSUPPORTED", "the cache is f16 or bf16"),
    (dict(heads=9), "SNL_E_UNSUPPORTED", "n_heads must be 1 to 64 times n_kv"),
    (dict(heads=130, kv=2), "SNL_E_UNSUPPORTED", "n_heads must be 1 to 64 times n_kv"),
])
def test_shapes_that_are_refused(lib, kw, kind, match):
    cache, batch, q = make(**kw)
    refused(kind, match, attend, cache, batch, q, work=16)
    lse = torch.zeros(q.shape[:2])
    refused(kind, match, cache.weigh, batch, q, lse)


def test_arguments_that_are_refused(lib):
    cache, batch, q = make()
    refused("SNL_E_INVALID", "work is too small", attend, cache, batch, q, work=0)
    refused("SNL_E_INVALID", "scale must be finite", attend, cache, batch, q, scale=float("nan"))
    refused("SNL_E_INVALID", "scale must be finite", attend, cache, batch, q, cap=-1.0)
    refused("SNL_E_INVALID", "q must be", attend, cache, batch, q[:2])
    refused("SNL_E_INVALID", "cache's type", attend, cache, batch, q.to(BF16))
    refused("SNL_E_INVALID", "first must be", attend, cache, batch, q, first=torch.zeros(3, dtype=torch.int64))
    refused("SNL_E_INVALID", "last must be", attend, cache, batch, q, last=torch.zeros(4, dtype=torch.int32))
    refused("SNL_E_INVALID", "slopes must be", attend, cache, batch, q, slopes=torch.zeros(4))
    refused("SNL_E_INVALID", "lse must be", attend, cache, batch, q, lse=torch.zeros(3, 8, dtype=F16))
    refused("SNL_E_INVALID", "gate must be", attend, cache, batch, q, gate=q[:, :4])
    wide = torch.zeros(3, 8, 260, dtype=F16)
    refused("SNL_E_INVALID", "aligned to 16 bytes", attend, cache, batch, wide[:, :, 4:])
    refused("SNL_E_INVALID", "aligned to 16 bytes", attend, cache, batch, q, out=wide[:, :, :256])
    refused("SNL_E_UNSUPPORTED", "tensors of float64", attend, cache, batch, q, out=q.double())
    lse = torch.zeros(3, 8)
    refused("SNL_E_INVALID", "decay must be finite", cache.weigh, batch, q, lse, decay=-0.5)
    refused("SNL_E_INVALID", "decay must be finite", cache.weigh, batch, q, lse, decay=float("inf"))
    bare, batch, q = make(weight=False)
    refused("SNL_E_INVALID", "no weights", bare.weigh, batch, q, lse)


def test_append_refusals(lib):
    cache, batch, q = make()
    k = torch.zeros(3, 2, 256, dtype=F16)
    pos = torch.zeros(3, 4, dtype=torch.int32)
    rope = torch.zeros(10, 32, 2)
    a = cache.append
    refused("SNL_E_UNSUPPORTED", "f32 or of the cache's type", a, batch, None, k.to(BF16), k.to(BF16), None)
    refused("SNL_E_INVALID", "one type", a, batch, None, k, k.float(), None)
    refused("SNL_E_INVALID", "cache's type", a, batch, q.float(), k.float(), k.float(), q.float())
    refused("SNL_E_INVALID", "pos be given", a, batch, q, k, k, q, None, rope)
    refused("SNL_E_INVALID", "pos must be", a, batch, q, k, k, q, pos[:, :3], rope)
    refused("SNL_E_INVALID", "add up to rot_dim / 2", a, batch, q, k, k, q, pos, rope, axes=paged.SECTIONS,
            sections=(11, 11, 11))
    refused("SNL_E_INVALID", "three axes", a, batch, q, k, k, q, pos, rope, sections=[11, 21])
    refused("SNL_E_INVALID", "unknown rotary layout", a, batch, q, k, k, q, pos, rope, axes=3)
    refused("SNL_E_UNSUPPORTED", "invalid rotary dim", a, batch, q, k, k, q, pos, torch.zeros(10, 129, 2))
    refused("SNL_E_INVALID", "q_norm must be", a, batch, q, k, k, q, q_norm=torch.zeros(128))
    for theta, rot in ((0.0, 64), (1e4, 258)):
        refused("SNL_E_INVALID", "theta must be positive", paged.rope_table, torch.zeros(4, rot // 2, 2), theta)


def test_evict_refusals(lib):
    cache, batch, q = make()
    kept = torch.zeros(1, 2, 8, dtype=torch.int32)
    into = torch.zeros(1, 1, dtype=torch.int32)
    lens = torch.zeros(1, dtype=torch.int32)
    refused("SNL_E_INVALID", "hold sink", cache.evict, batch, 8, kept, sink=5, recent=4)
    refused("SNL_E_INVALID", "kept must be", cache.evict, batch, 9, kept)
    refused("SNL_E_INVALID", "budget must be positive", cache.evict, batch, 0, kept[:, :, :0])
    refused("SNL_E_INVALID", "new_lens is needed", cache.evict, batch, 8, kept, into)
    refused("SNL_E_INVALID", "into must be", cache.evict, batch, 8, kept, into.long(), lens)
    cache, batch, q = make(page=8)
    kept = torch.zeros(1, 2, 9, dtype=torch.int32)
    refused("SNL_E_INVALID", "do not hold the budget", cache.evict, batch, 9, kept, into, lens)
    bare, batch, q = make(weight=False)
    refused("SNL_E_INVALID", "no weights", bare.evict, batch, 9, kept)


def test_null_arguments(lib):
    cache, batch, q = make()
    for rc in (lib.snl_paged_append(None, None, None, *[None] * 9), lib.snl_paged_attend(None, None, None, *[None] * 5, 0, None),
               lib.snl_paged_weigh(None, None, None, None, None, 1.0, None),
               lib.snl_paged_evict(None, None, None, None, None, None, None),
               lib.snl_paged_append(cache.ref, batch.ref, None, *[None] * 9),
               lib.snl_paged_attend(cache.ref, batch.ref, C.byref(ffi.PagedAttnP()), *[None] * 5, 0, None),
               lib.snl_rope_table(1e4, 64, 4, None, None)):
        assert rc == -1 and b"null" in lib.snl_last_error()
    assert lib.snl_paged_attend_workspace(None, None, 1) == 0


def test_batch_and_cache_shapes(lib):
    k = torch.zeros(4, 2, 16, 256, dtype=F16)
    with pytest.raises(SnlError, match="same shape"):
        paged.PagedCache(k, k.transpose(1, 2).contiguous().transpose(1, 2))
    with pytest.raises(SnlError, match="contiguous"):
        paged.PagedCache(k[..., ::2], k[..., ::2])
    with pytest.raises(SnlError, match="weight must be"):
        paged.PagedCache(k, k.clone(), torch.zeros(4, 16, 2))
    with pytest.raises(SnlError, match="start must be"):
        paged.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                         torch.zeros(2, dtype=torch.int32), 1, 1)


def test_struct_sizes(lib):
    assert [C.sizeof(s) for s in (ffi.PagedCacheC, ffi.PagedBatchC, ffi.PagedAppendP, ffi.PagedAttnP, ffi.PagedEvictP)] == \
        [72, 40, 104, 96, 16]


def test_numbers_that_no_field_holds(lib):
    cache, batch, q = make()
    for kw in (dict(window=-1), dict(window=1 << 32), dict(window=1.5), dict(scale=1e39), dict(cap="soft")):
        refused("SNL_E_INVALID", "the attention's numbers|scale must be finite", attend, cache, batch, q, **kw)
    new = torch.zeros(3, 2, 256)
    for kw in (dict(axes=-1), dict(sections=(1 << 32, 0, 0)), dict(sections=(0, -1, 0)), dict(eps=1e39)):
        refused("SNL_E_INVALID", "append's numbers|eps must be finite", cache.append, batch, None, new, new, None, **kw)


def test_rope_table_alignment(lib):
    """Its pairs are written eight bytes at a time."""
    table = torch.zeros(4 * 32 * 2 + 1)[1:].view(4, 32, 2)
    assert table.data_ptr() % 8 == 4
    refused("SNL_E_INVALID", "aligned to 8 bytes", paged.rope_table, table, 1e4)


def test_numbers_that_no_field_of_batch_or_evict_holds(lib):
    cache, batch, q = make()
    kept = torch.zeros(1, 2, 8, dtype=torch.int32)
    for kw in (dict(sink=(1 << 32) + 1), dict(recent=1 << 32), dict(sink=-1), dict(recent=1.5)):
        refused("SNL_E_INVALID", "evict's numbers", cache.evict, batch, 8, kept, **kw)
    for budget in ((1 << 32) + 8, -1, 8.0):
        refused("SNL_E_INVALID", "evict's numbers", cache.evict, batch, budget, kept)
    for rows, longest in ((3, (1 << 32) + 9), (3, -1), (3, 9.0), ((1 << 32) + 3, 9), (-1, 9), ("3", 9)):
        refused("SNL_E_INVALID", "the batch's numbers", paged.PagedBatch, *batch.tensors, rows, longest)


def test_batch_without_sequences(lib):
    """Nothing to do is done, though tensors without elements have no address."""
    cache, _, _ = make()
    ints = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    batch = paged.PagedBatch(ints(0, 4), ints(1), ints(0), 0, 9)
    q, k = torch.zeros(0, 8, 256, dtype=F16), torch.zeros(0, 2, 256, dtype=F16)
    cache.append(batch, q, k, k, torch.zeros_like(q))
    attend(cache, batch, q, lse=torch.zeros(0, 8))
    cache.weigh(batch, q, torch.zeros(0, 8))
    cache.evict(batch, 8, ints(0, 2, 8))
    cache.evict(batch, 8, ints(0, 2, 8), ints(0, 1), ints(0))


def test_tables_without_an_address(lib):
    """A batch with sequences needs its arrays."""
    cache, batch, q = make()
    for field in ("table", "start", "len"):
        b = ffi.PagedBatchC.from_buffer_copy(batch.c)
        setattr(b, field, None)
        rc = lib.snl_paged_weigh(cache.ref, C.byref(b), C.byref(ffi.PagedAttnP()), None, None, 1.0, None)
        assert rc == -1 and b"null array" in lib.snl_last_error()
    kept = torch.zeros(1, 2, 8, dtype=torch.int32)
    p = ffi.PagedEvictP(8, 0, 0, 0)
    for args in ((None, None, batch.c.len), (kept.data_ptr(), None, None)):
        assert lib.snl_paged_evict(cache.ref, batch.ref, p, *args, None) == -1 and b"null argument" in lib.snl_last_error()


def test_scratch_that_is_not_there(lib):
    """The bytes of a view count only where they lie together."""
    cache, batch, q = make()
    need = cache.attend_workspace(batch, 8)
    for work in (torch.zeros(1, dtype=torch.uint8).expand(need), torch.zeros(2 * need, dtype=torch.uint8)[::2]):
        refused("SNL_E_INVALID", "work must be contiguous", cache.attend, batch, q, torch.zeros_like(q), work)


def test_outputs_over_one_another(lib):
    """Rows or heads of an output at one place would be written in no order."""
    cache, batch, q = make()
    new = torch.zeros(3, 2, 256, dtype=F16)
    for view in (torch.zeros(1, 8, 256, dtype=F16).expand(3, 8, 256), torch.zeros(3, 1, 256, dtype=F16).expand(3, 8, 256),
                 torch.zeros(8192, dtype=F16).as_strided((3, 8, 256), (2048, 128, 1))):
        refused("SNL_E_INVALID", "out overlap", attend, cache, batch, q, out=view)
        refused("SNL_E_INVALID", "q_out overlap", cache.append, batch, q, new, new, view)
