"""The paged-cache operators on the GPU against their definitions in 64 bits."""
import math

import pytest

from sensenova_b200 import ffi, paged

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
import paged_ref as ref  # noqa: E402
from paged_ref import Problem  # noqa: E402

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _clean(torch_cuda, lib):
    torch.cuda.synchronize()
    lib.snl_device_error(1)
    yield
    torch.cuda.synchronize()
    assert lib.snl_device_error(1) == 0


def run_attend(p, q=None, gate=None, out_dtype=None, lse=True, stream=0, **masks):
    q = p.q if q is None else q
    cache, batch = p.cache(paged), p.batch(paged)
    out = torch.full((p.n, p.heads, p.d), math.nan, dtype=out_dtype or p.dtype, device="cuda")
    z = torch.full((p.n, p.heads), math.nan, device="cuda") if lse else None
    work = torch.full((cache.attend_workspace(batch, p.heads),), 0xAB, dtype=torch.uint8, device="cuda")
    cache.attend(batch, q, out, work, lse=z, gate=gate, stream=stream, **masks)
    return out, z


def check_attend(p, q=None, gate=None, out_dtype=None, **masks):
    q = p.q if q is None else q
    out, lse = run_attend(p, q, gate, out_dtype, **masks)
    want, z, tol, ltol = ref.attend(p, q, gate, out_dtype=out_dtype, **masks)
    assert torch.equal(torch.isneginf(lse), torch.isneginf(z))
    assert ((lse.double() - z).abs().nan_to_num(0) <= ltol).all()
    off = (out.double() - want).abs() - tol
    assert (off <= 0).all(), float(off.max())
    return out, lse


SHAPES = [  # heads, kv, d, page, layout, type
    (4, 1, 256, 16, "head", F16), (16, 4, 256, 64, "slot", F16), (32, 8, 128, 32, "head", BF16),
    (6, 2, 256, 8, "slot", BF16), (20, 4, 128, 128, "head", F16), (8, 8, 256, 16, "slot", BF16),
    (32, 1, 128, 16, "slot", F16), (64, 1, 256, 256, "head", F16),
]


@pytest.mark.parametrize("heads,kv,d,page,layout,dtype", SHAPES)
@pytest.mark.parametrize("lens,rows", [
    ([1], [1]), ([129], [1]), ([7, 300, 64, 1], [1, 1, 1, 1]), ([40], [40]), ([500, 63, 130], [37, 63, 2]),
])
def test_attend_shapes(heads, kv, d, page, layout, dtype, lens, rows):
    check_attend(Problem(lens, rows, heads, kv, d, page, layout, dtype, seed=len(lens) + heads))


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 127, 128, 129, 255, 256, 257, 1000])
@pytest.mark.parametrize("rows", [1, 31, 33])
def test_attend_lengths(n, rows):
    check_attend(Problem([n], [min(rows, n)], seed=n))


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("rows", [1, 70])
def test_attend_long(d, rows):
    """Keys split over the GPU and joined; the sums over keys are longer, so is their share."""
    p = Problem([5000, 9000, 130], [rows, rows, 1], 8, 2, d, 64, seed=d)
    check_attend(p)


MASKS = {
    "cap": dict(cap=5.0),
    "slopes": dict(slopes=True),
    "window": dict(window=50),
    "window 1": dict(window=1),
    "docs": dict(docs=70),
    "blocks": dict(block=48),
    "prefix": dict(prefix=90),
    "empty rows": dict(empty=True),
    "all": dict(cap=20.0, slopes=True, window=100, docs=130, block=30, empty=True),
    "scale": dict(scale=-0.11),
}


def masks_of(p, cap=0.0, slopes=False, window=0, docs=0, block=0, prefix=0, empty=False, scale=None):
    t = p.slot()
    first = last = None
    if docs:
        first = t // docs * docs
    if empty:
        first = torch.zeros_like(t) if first is None else first
        first = torch.where(torch.arange(len(t)) % 5 == 2, 2**31 - 1, first)
    if block:
        last = (t // block + 1) * block
    if prefix:
        last = torch.full_like(t, prefix)
    m = dict(cap=cap, window=window)
    if slopes:
        m["slopes"] = torch.tensor([2.0 ** (-8 * (h + 1) / p.heads) for h in range(p.heads)], device="cuda")
    if first is not None:
        m["first"] = first.to(torch.int32).cuda()
    if last is not None:
        m["last"] = last.to(torch.int32).cuda()
    if scale is not None:
        m["scale"] = scale
    return m


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("d,rows", [(256, [37, 150, 1]), (128, [37, 150, 1]), (256, [1, 1, 1])])
def test_attend_masks(mask, d, rows):
    p = Problem([300, 150, 77], rows, 8, 2, d, 16, seed=d + rows[0])
    check_attend(p, **masks_of(p, **MASKS[mask]))


@pytest.mark.parametrize("rows", [[70, 1], [1, 1]])
def test_attend_nothing_seen(rows):
    p = Problem([200, 40], rows, seed=3)
    out, lse = run_attend(p, first=torch.full((p.n,), 2**31 - 1, dtype=torch.int32, device="cuda"))
    assert (out == 0).all() and torch.isneginf(lse).all()


def test_attend_empty_sequences():
    """Sequences without rows, without slots, and a batch without rows."""
    p = Problem([0, 40, 300, 0, 17], [0, 0, 33, 0, 1], 8, 2, seed=4)
    check_attend(p)
    p = Problem([0, 40], [0, 0], seed=4)
    out, lse = run_attend(p)
    assert out.shape[0] == 0


@pytest.mark.parametrize("rows", [1, 100])
def test_attend_hides_what_is_not_seen(rows):
    """NaN and infinities in keys and values that a row does not see leave it as it is: before
    the window, before the document, after its own slot (where later rows do see them)."""
    p = Problem([400], [rows], 8, 2, seed=5)
    pg, sl = p.where(0)
    m = masks_of(p, window=90)
    clean, _ = run_attend(p, **m)
    low = 400 - rows - 89  # below every row's window
    p.k[pg[:low - 1], :, sl[:low - 1]] = math.inf
    p.v[pg[:low - 1], :, sl[:low - 1]] = math.nan
    p.v[pg[low - 1], 0, sl[low - 1], 7] = -math.inf
    assert torch.equal(run_attend(p, **m)[0], clean)
    if rows > 1:
        at = 360  # rows 0..59 are before it
        for bad in (math.nan, math.inf):
            p.v[pg[at], 1, sl[at], 9] = bad
            out, _ = run_attend(p, **m)
            assert torch.equal(out[:60], clean[:60])
            same = torch.ones(8, 256, dtype=torch.bool)
            same[4:, 9] = False
            assert torch.equal(out[60:][:, same], clean[60:][:, same])
            hit = out[60:, 4:, 9]
            assert (hit.isnan() if math.isnan(bad) else hit == math.inf).all()
        p.k[pg[at], 0, sl[at], 3] = math.nan
        out, _ = run_attend(p, **m)
        assert torch.equal(out[:60], clean[:60]) and out[60:, :4].isnan().all()


def test_attend_nan_in_own_rows():
    """A NaN query gives NaN in its own row and head only."""
    p = Problem([300], [64], 8, 2, seed=6)
    clean, z = run_attend(p)
    q = p.q.clone()
    q[10, 3, 5] = math.nan
    out, lse = run_attend(p, q)
    assert out[10, 3].isnan().all() and lse[10, 3].isnan()
    keep = torch.ones(64, 8, dtype=torch.bool)
    keep[10, 3] = False
    assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], z[keep])


@pytest.mark.parametrize("size", [1e-4, 60.0, 3e3])
def test_attend_large_and_small_scores(size):
    """Scores near zero, scores that leave one key, and scores of thousands."""
    p = Problem([333], [45], 4, 1, seed=7, peak=1.0)
    q = (p.q.float() * size).to(F16)
    check_attend(p, q)


@pytest.mark.parametrize("gate_dtype", [F16, F32])
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_strides_gate_types(gate_dtype, rows):
    """q, gate and out as parts of wider rows; f32 gate and out."""
    p = Problem([200, 90], [rows, rows], 8, 2, seed=8)
    wide = p.normal(p.n, 8, 2, 264).to(F16)
    q = wide[:, :, 0, 8:]
    gate = p.normal(p.n, 8, 512).to(gate_dtype)[:, :, 256:]
    check_attend(p, q, gate)
    cache, batch = p.cache(paged), p.batch(paged)
    out = torch.full((8, p.n, 260), math.nan, device="cuda").transpose(0, 1)
    work = torch.empty(cache.attend_workspace(batch, 8), dtype=torch.uint8, device="cuda")
    cache.attend(batch, q, out[:, :, :256], work, gate=gate)
    want, _, tol, _ = ref.attend(p, q, gate, out_dtype=F32)
    assert ((out[:, :, :256].double() - want).abs() <= tol).all()
    assert out[:, :, 256:].isnan().all()


@pytest.mark.parametrize("rows", [1, 50])
def test_attend_same_bits_every_time(rows):
    p = Problem([3000, 700], [rows, rows], 8, 2, seed=9)
    a, z = run_attend(p)
    for _ in range(3):
        b, y = run_attend(p)
        assert torch.equal(a, b) and torch.equal(z, y)


@pytest.mark.parametrize("d,rows", [(256, 1), (256, 40), (128, 40)])
def test_attend_other_stream_and_graph(d, rows):
    p = Problem([1500, 64], [rows, rows], 8, 2, d, seed=10)
    a, _ = run_attend(p)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b, _ = run_attend(p, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(a, b)
    cache, batch = p.cache(paged), p.batch(paged)
    out = torch.zeros_like(a)
    work = torch.empty(cache.attend_workspace(batch, 8), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        cache.attend(batch, p.q, out, work, stream=torch.cuda.current_stream().cuda_stream)
    p.len_t[0] -= 5  # lengths are the device's: a replay sees the new ones
    p.lens[0] -= 5
    g.replay()
    want, _, tol, _ = ref.attend(p, p.q)
    assert ((out.double() - want).abs() <= tol).all()


def test_attend_far_pages():
    """Pages past 2^32 elements of the pool."""
    pages = 2**32 // (64 * 256) + 40
    p = Problem([200], [20], 4, 1, 256, 64, seed=11)
    k, v = (torch.empty(pages, 1, 64, 256, dtype=F16, device="cuda") for _ in range(2))
    at = [pages - 1 - 3 * i for i in range(len(p.pages[0]))]
    k[at], v[at] = p.k[p.pages[0]], p.v[p.pages[0]]
    want, _ = run_attend(p)
    p.k, p.v, p.pages = k, v, [at]
    p.table = torch.tensor([at], dtype=torch.int32, device="cuda")
    got, _ = run_attend(p)
    assert torch.equal(got, want)


def test_bad_indices_are_reported(lib):
    """A page outside the cache and a length over max_len set bit 2, and leave other sequences alone."""
    p = Problem([100, 100], [20, 20], 8, 2, seed=12)
    want, _ = run_attend(p)
    p.table[0, 2] = 10**6
    got, _ = run_attend(p)
    torch.cuda.synchronize()
    assert lib.snl_device_error(1) == 4 and torch.equal(got[20:], want[20:])
    p.table[0, 2] = p.pages[0][2]
    p.len_t[0] = 500
    got, _ = run_attend(p)
    torch.cuda.synchronize()
    assert lib.snl_device_error(1) == 4 and torch.equal(got[20:], want[20:])


@pytest.mark.parametrize("page", [8, 16, 128])
@pytest.mark.parametrize("d,lens,rows", [(256, [1000, 700], [70, 3]), (128, [1000, 700], [70, 3]), (256, [9000], [40]),
                                         (128, [1000, 700], [1, 1])])
def test_attend_pages_that_no_row_sees(d, lens, rows, page):
    """Pages wholly before every row's window may be gone from the table: nothing changes, nothing is reported."""
    p = Problem(lens, rows, 8, 2, d, page, seed=page)
    m = masks_of(p, window=90)
    want, z = check_attend(p, **m)
    for i, n in enumerate(lens):
        p.table[i, :(n - rows[i] - 89) // page] = -1
    out, lse = run_attend(p, **m)
    assert torch.equal(out, want) and torch.equal(lse, z)


@pytest.mark.parametrize("d,rows", [(128, 1), (256, 1), (128, 3), (256, 3)])
def test_attend_many_sequences(d, rows):
    """More sequences than one look at 32 boundaries finds, lengths of every kind."""
    lens = [max(rows, (i * 37) % 90) if i % 11 else 0 for i in range(260)]
    p = Problem(lens, [min(n, rows) for n in lens], 8, 2, d, 8, seed=d + rows)
    check_attend(p)
    check_attend(p, **masks_of(p, window=20, slopes=True))


@pytest.mark.parametrize("d", [128, 256])
def test_attend_uneven_rows(d):
    """At most two rows a sequence on the average, many in one; two rows in each."""
    check_attend(Problem([300, 70, 5, 90, 64, 1, 33], [9, 1, 0, 1, 1, 1, 1], 8, 2, d, seed=1))
    check_attend(Problem([300, 70, 5, 900], [2, 2, 2, 2], 8, 1, d, seed=2), window=200)
    check_attend(Problem([30000, 21000], [2, 1], 32, 8, d, 64, seed=25))  # more blocks than the few-row kernel takes at 256
    check_attend(Problem([40, 130], [2, 1], 6, 2, d, seed=3), cap=9.0)


@pytest.mark.parametrize("rows", [1, 50])
def test_attend_zero_scale(rows):
    """Equal scores: the mean of the values."""
    p = Problem([333], [rows], 4, 1, seed=19)
    check_attend(p, scale=0.0)


@pytest.mark.parametrize("rows", [1, 40])
def test_attend_generous_bounds(rows):
    """max_len and the table's rows far past the lengths: parts that no sequence reaches."""
    p = Problem([200, 64, 900], [rows] * 3, 8, 2, seed=20, width=3000, max_len=40000)
    check_attend(p)


@pytest.mark.parametrize("rows", [1, 40])
def test_pages_inside_a_wider_pool(rows):
    """k and v as the halves of one tensor per page, two layers deep."""
    p = Problem([200, 77], [rows, rows], 8, 2, 256, 16, seed=21, weight=True)
    want, lse = run_attend(p)
    pool = torch.full((p.k.shape[0], 2, 2, 2, 16, 264), math.nan, dtype=F16, device="cuda")
    k, v = pool[:, 1, 0, :, :, :256], pool[:, 1, 1, :, :, :256]
    k.copy_(p.k), v.copy_(p.v)
    p.k, p.v = k, v
    got, z = run_attend(p)
    assert torch.equal(got, want) and torch.equal(z, lse)
    check_weigh(p)


# ---- append --------------------------------------------------------------------------------


@pytest.mark.parametrize("heads,kv,d,page,layout,dtype", SHAPES)
@pytest.mark.parametrize("axes,pairs,rot,normed,src", [
    (paged.INTERLEAVED, paged.HALVES, 64, True, F32), (paged.SECTIONS, paged.ADJACENT, 64, False, None),
    (paged.ONE, paged.HALVES, 128, True, None), (paged.SECTIONS, paged.HALVES, 10, True, F32), (paged.ONE, 0, 0, True, F32),
])
def test_append(heads, kv, d, page, layout, dtype, axes, pairs, rot, normed, src):
    lens, rows = [37, 1, 200, 9], [5, 1, 131, 9]
    p = Problem(lens, rows, heads, kv, d, page, layout, dtype, seed=rot + heads)
    src = src or dtype
    n = p.n
    wide = p.normal(n, (2 * heads + 2 * kv) * d).to(src)  # per head [q | gate], then k, then v
    q = wide[:, :2 * heads * d].view(n, heads, 2 * d)[:, :, :d]
    k = wide[:, 2 * heads * d:(2 * heads + kv) * d].view(n, kv, d)
    v = wide[:, (2 * heads + kv) * d:].view(n, kv, d)
    qn, kn = (0.2 * p.normal(d), 0.2 * p.normal(d)) if normed else (None, None)
    half = rot // 2
    sections = (half - 2 * (half // 3), half // 3, half // 3)
    pos = torch.randint(0, 5000, (n, 4), generator=p.gen, device="cuda", dtype=torch.int32)
    rope = None
    if rot:
        rope = torch.empty(5000, half, 2, device="cuda")
        paged.rope_table(rope, 1e7)
    before = p.k.clone(), p.v.clone()
    q_out = torch.empty(n, heads, d, dtype=dtype, device="cuda")
    p.cache(paged).append(p.batch(paged), q, k, v, q_out, pos if rot else None, rope, axes=axes, pairs=pairs,
                          sections=sections, q_norm=qn, k_norm=kn)
    u = ref.UNIT[dtype]

    def near(got, want, size):  # one rounding, and a few of 32 bits in the norm and the turn
        return ((got.double() - want).abs() <= u * want.abs() + 16 * 2.0**-24 * size + ref.TINY[dtype]).all()

    want = ref.turned(q, pos, rope, axes, pairs, sections, qn)
    assert near(q_out, want, want.abs().amax(-1, keepdim=True))
    want = ref.turned(k, pos, rope, axes, pairs, sections, kn)
    fresh = torch.zeros(p.k.shape[0], page, dtype=torch.bool, device="cuda")
    for i in range(len(lens)):
        r0, r1 = p.seq_rows(i)
        pg, sl = p.where(i)
        pg, sl = pg[lens[i] - rows[i]:], sl[lens[i] - rows[i]:]
        fresh[pg, sl] = True
        assert near(p.k[pg, :, sl], want[r0:r1], want[r0:r1].abs().amax(-1, keepdim=True))
        assert torch.equal(p.v[pg, :, sl], v[r0:r1].to(dtype))
    for now, was in zip((p.k, p.v), before):  # nothing else is written
        now, was = (x.transpose(1, 2)[~fresh].nan_to_num(77) for x in (now, was))
        assert torch.equal(now, was)


def test_append_without_q_and_other_stream():
    p = Problem([20, 33], [4, 33], 4, 2, seed=1)
    k, v = p.normal(p.n, 2, 256).to(F16), p.normal(p.n, 2, 256).to(F16)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    p.cache(paged).append(p.batch(paged), None, k, v, None, stream=s.cuda_stream)
    s.synchronize()
    pg, sl = p.where(1)
    assert torch.equal(p.k[pg, :, sl], k[4:]) and torch.equal(p.v[pg, :, sl], v[4:])


def test_rope_table_far_positions():
    t = torch.empty(262144, 32, 2, device="cuda")
    paged.rope_table(t, 1e7)
    f = torch.arange(32, dtype=torch.float64, device="cuda")
    a = torch.arange(262144, dtype=torch.float64, device="cuda")[:, None] * 1e7 ** (-2 * f / 64)
    # one rounding to 32 bits, and 64-bit angles off by a few 2^-53 of up to 262144
    assert ((t[..., 0].double() - a.cos()).abs() <= 2.0**-24).all()
    assert ((t[..., 1].double() - a.sin()).abs() <= 2.0**-24).all()


def test_append_reports_positions(lib):
    p = Problem([5], [5], 4, 1, seed=2)
    x = p.normal(5, 1, 256).to(F16)
    pos = torch.tensor([[3, 0, 0, 0]] * 4 + [[40, 0, 0, 0]], dtype=torch.int32, device="cuda")
    rope = torch.zeros(40, 16, 2, device="cuda")
    p.cache(paged).append(p.batch(paged), None, x, x, None, pos, rope)
    torch.cuda.synchronize()
    assert lib.snl_device_error(1) == 4


# ---- weigh ---------------------------------------------------------------------------------


def check_weigh(p, decay=1.0, **masks):
    _, lse, _, _ = ref.attend(p, p.q, **masks)
    lse = lse.float()
    want, tol = ref.weigh(p, p.q, lse, p.weight, decay, **masks)
    p.cache(paged).weigh(p.batch(paged), p.q, lse, decay=decay, **masks)
    got = p.weight.double()
    assert torch.equal(got.isnan(), want.isnan())
    off = ((got - want).abs() - tol).nan_to_num(0)
    assert (off <= 0).all(), float(off.max())


@pytest.mark.parametrize("heads,kv,d,page,layout,dtype", SHAPES)
@pytest.mark.parametrize("lens,rows", [([1], [1]), ([7, 300, 64], [1, 1, 1]), ([500, 63, 130], [37, 63, 2])])
def test_weigh_shapes(heads, kv, d, page, layout, dtype, lens, rows):
    check_weigh(Problem(lens, rows, heads, kv, d, page, layout, dtype, seed=heads, weight=True))


@pytest.mark.parametrize("n", [1, 2, 127, 128, 129, 257])
@pytest.mark.parametrize("decay", [0.0, 0.5])
def test_weigh_lengths(n, decay):
    check_weigh(Problem([n, 40], [min(n, 33), 1], seed=n, weight=True), decay)


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("d,rows", [(256, [37, 150, 1]), (128, [1, 1, 1])])
def test_weigh_masks(mask, d, rows):
    p = Problem([300, 150, 77], rows, 8, 2, d, 16, seed=d, weight=True)
    check_weigh(p, **masks_of(p, **MASKS[mask]))


def test_weigh_hides_what_is_not_seen():
    """Old weights of the step's own slots, NaN keys that no row sees, sequences without rows."""
    p = Problem([300, 60, 0], [64, 0, 0], 8, 2, seed=13, weight=True)
    pg, sl = p.where(0)
    p.weight[pg[236:], :, sl[236:]] = math.nan
    m = masks_of(p, window=50)
    check_weigh(p, **m)
    p.k[pg[:100], :, sl[:100]] = math.nan
    before = p.weight.clone()
    _, lse = run_attend(p, **m)
    p.cache(paged).weigh(p.batch(paged), p.q, lse, **m)
    assert torch.equal(p.weight[pg[:100], :, sl[:100]], before[pg[:100], :, sl[:100]])
    assert not p.weight[pg, :, sl].isnan().any()


@pytest.mark.parametrize("heads", [33, 40, 17, 64])
@pytest.mark.parametrize("rows", [1, 5])
def test_weigh_large_groups(heads, rows):
    """Heads of one KV head that do not divide a tile, or fill more than half of one."""
    check_weigh(Problem([150, 300], [rows, 21 if rows > 1 else 1], heads, 1, 128, seed=heads, weight=True))


@pytest.mark.parametrize("d,rows", [(128, 1), (256, 1), (128, 3), (256, 3)])
def test_weigh_many_sequences(d, rows):
    lens = [max(rows, (i * 37) % 90) if i % 11 else 0 for i in range(150)]
    check_weigh(Problem(lens, [min(n, rows) for n in lens], 8, 2, d, 8, seed=d + rows, weight=True), 0.5)


@pytest.mark.parametrize("d", [128, 256])
def test_weigh_uneven_rows(d):
    check_weigh(Problem([300, 70, 5, 90, 64, 1, 33], [9, 1, 0, 1, 1, 1, 1], 8, 2, d, seed=1, weight=True))
    check_weigh(Problem([300, 70, 5, 900], [2, 2, 2, 2], 8, 1, d, seed=2, weight=True), window=200, cap=20.0)


def test_weigh_long():
    check_weigh(Problem([3000, 2100], [700, 1], 8, 2, 256, 64, seed=22, weight=True), 0.9)


@pytest.mark.parametrize("heads", [8, 9, 16, 40, 64])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("decay", [0.0, 0.5])
def test_weigh_without_rows(heads, d, decay):
    """The weights decay, whatever the number of heads to a KV head."""
    check_weigh(Problem([150, 300, 0, 1], [0, 0, 0, 0], heads, 1, d, seed=heads, weight=True), decay)


def test_weigh_sums_to_the_rows():
    """Every row hands out a weight of one per head."""
    p = Problem([700], [90], 8, 2, seed=14, weight=True)
    _, lse = run_attend(p)
    p.cache(paged).weigh(p.batch(paged), p.q, lse, decay=0.0)
    pg, sl = p.where(0)
    total = p.weight[pg, :, sl].double().sum(0)
    assert ((total - 90 * 4).abs() <= 90 * 4 * 2e-5).all()


# ---- evict ---------------------------------------------------------------------------------


def check_evict(p, budget, sink, recent, in_place, extra_pages=0):
    kept = torch.full((len(p.lens), p.kv, budget), 99, dtype=torch.int32, device="cuda")
    k, v, w = p.k.clone(), p.v.clone(), p.weight.clone()
    cache, batch = p.cache(paged), p.batch(paged)
    if in_place:
        new_lens, to = p.len_t, p.pages
        cache.evict(batch, budget, kept, sink=sink, recent=recent)
    else:
        n = -(-budget // p.page)
        to = [p.free[i * n:(i + 1) * n] for i in range(len(p.lens))]
        into = torch.tensor(to, dtype=torch.int32, device="cuda")
        new_lens = torch.empty_like(p.len_t)
        cache.evict(batch, budget, kept, into, new_lens, sink=sink, recent=recent)
    assert new_lens.tolist() == [min(n, budget) for n in p.lens]
    for i, n in enumerate(p.lens):
        pg, sl = p.where(i)
        at = torch.arange(min(n, budget))
        ng, ns = torch.tensor(to[i], dtype=torch.long)[at // p.page].cuda(), (at % p.page).cuda()
        old = w[pg, :, sl].cpu()
        for h in range(p.kv):
            want = ref.evict(old[:, h].tolist(), n, budget, sink, recent)
            assert kept[i, h].tolist() == want + [-1] * (budget - len(want))
            src = torch.tensor(want, dtype=torch.long, device="cuda")
            for now, was in ((p.k, k), (p.v, v), (p.weight, w)):
                a, b = now[ng, h, ns], was[pg[src], h, sl[src]]
                assert torch.equal(a.nan_to_num(55), b.nan_to_num(55))
    if not in_place:  # the old pages are as they were
        mine = [x for s in p.pages for x in s]
        assert torch.equal(p.k[mine].nan_to_num(55), k[mine].nan_to_num(55))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([100, 30, 1, 0, 64], 64, 4, 16), ([1000, 1100], 512, 0, 0), ([300], 299, 4, 64), ([300], 1, 0, 0),
    ([300], 300, 4, 4), ([300], 80, 16, 64), ([2500, 40], 1031, 1, 1), ([9], 8, 8, 0), ([9], 8, 0, 8),
])
@pytest.mark.parametrize("kv,d,page,layout", [(1, 256, 16, "head"), (3, 128, 32, "slot")])
def test_evict(lens, budget, sink, recent, in_place, kv, d, page, layout):
    p = Problem(lens, [min(n, 1) for n in lens], 4 * kv, kv, d, page, layout, seed=budget, weight=True,
                spare=len(lens) * -(-budget // page))
    check_evict(p, budget, sink, recent, in_place)


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("values", ["ties", "zeros", "odd"])
def test_evict_ties_and_odd_weights(values, in_place):
    """Equal weights keep the lowest slots; -0 and 0 are equal; NaN counts as -inf."""
    p = Problem([400, 777], [1, 1], 8, 2, seed=15, weight=True, spare=50)
    if values == "ties":
        p.weight = (p.weight * 6).round()
    elif values == "zeros":
        p.weight = torch.where(p.weight > 0.5, 0.0, -0.0)
    else:
        x = p.weight
        pick = (x * 1000).nan_to_num(0).long() % 6
        p.weight = torch.stack([x, x - 0.5, x * 1e-42, torch.full_like(x, math.inf), torch.full_like(x, -math.inf),
                                torch.full_like(x, math.nan)])[pick, *torch.meshgrid(*[torch.arange(n, device="cuda") for n in x.shape], indexing="ij")]
    check_evict(p, 350, 2, 30, in_place)


@pytest.mark.parametrize("budget", [1000, 57000])
def test_evict_long(budget):
    """More candidates than shared memory holds keys of."""
    p = Problem([60000], [1], 2, 1, 128, 64, seed=23, weight=True, spare=-(-budget // 64))
    check_evict(p, budget, 4, 64, False)


def test_evict_many_sequences():
    lens = [(i * 53) % 200 for i in range(70)]
    p = Problem(lens, [min(n, 1) for n in lens], 4, 2, 128, 8, seed=24, weight=True, spare=70 * 8)
    check_evict(p, 60, 2, 10, False)


# ---- together --------------------------------------------------------------------------------


def test_serving_a_prompt_in_chunks_equals_one_chunk():
    """append + attend in chunks and single tokens give what one chunk gives."""
    p = Problem([150], [150], 8, 2, seed=16)
    x = [p.normal(150, h, 256).to(F16) for h in (8, 2, 2)]
    pos = torch.arange(150, dtype=torch.int32, device="cuda")[:, None].repeat(1, 4).contiguous()
    rope = torch.empty(200, 32, 2, device="cuda")
    paged.rope_table(rope, 1e4)
    q_out = torch.empty(150, 8, 256, dtype=F16, device="cuda")
    p.cache(paged).append(p.batch(paged), *x, q_out, pos, rope)
    whole, _, tol, _ = ref.attend(p, q_out)
    p.k.fill_(math.nan), p.v.fill_(math.nan)
    got, at = [], 0
    for n in (64, 1, 1, 70, 14):
        p.lens, p.rows, p.n = [at + n], [n], n
        p.len_t.fill_(at + n)
        p.start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        s = slice(at, at + n)
        out = torch.empty(n, 8, 256, dtype=F16, device="cuda")
        p.cache(paged).append(p.batch(paged), *(y[s] for y in x), out, pos[s].contiguous(), rope)
        assert torch.equal(out, q_out[s])
        got.append(run_attend(p, out)[0])
        at += n
    assert ((torch.cat(got).double() - whole).abs() <= tol).all()


def test_evicted_cache_attends_like_its_kept_slots():
    """attend -> weigh -> evict -> attend of the next token sees the kept slots of each head."""
    p = Problem([600], [100], 8, 2, seed=17, weight=True, spare=20)
    _, lse = run_attend(p)
    cache, batch = p.cache(paged), p.batch(paged)
    cache.weigh(batch, p.q, lse, decay=0.0)
    kept = torch.empty(1, 2, 256, dtype=torch.int32, device="cuda")
    k, v = (p.keys(0, x) for x in (p.k, p.v))
    cache.evict(batch, 256, kept, sink=4, recent=32)
    assert int(p.len_t[0]) == 256
    p.lens, p.rows, p.n = [256], [1], 1
    p.start = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    p.q = p.q[-1:]
    out, lse = check_attend(p)
    for h in range(2):
        i = kept[0, h].long()
        s = p.q[0, 4 * h:4 * h + 4].double() @ k[i, h].T / 16
        want = torch.softmax(s, -1) @ v[i, h]
        assert ((out[0, 4 * h:4 * h + 4].double() - want).abs() <= 4e-3).all()  # 8 roundings of 2^-11 of values up to 1


def test_matches_the_contiguous_cache(lib):
    """append and attend over pages against snl_attn_prep and snl_attend over the engine's cache."""
    import ctypes as C

    from sensenova_b200.ffi import AttnP, StepU

    n, heads, kv = 96, 16, 4
    p = Problem([n], [n], heads, kv, seed=18)
    proj = p.normal(n, (2 * heads + 2 * kv) * 256)
    norms = 0.1 * p.normal(512)
    pos = torch.randint(0, 3000, (n, 4), generator=p.gen, device="cuda", dtype=torch.int32)
    ap = AttnP(heads, kv, 64, proj.shape[1], 1e7, 1e-6, 1 / 16.0, (33 << 16) | 30)
    st = StepU(n, 0, 1, 0)
    ptr = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    qbuf = torch.empty(n, heads * 256, device="cuda")
    kc, vc = (torch.empty(n * kv * 256, dtype=F16, device="cuda") for _ in range(2))
    want = torch.empty(n, heads * 256, device="cuda")
    ffi.check(lib.snl_attn_prep(C.byref(st), C.byref(ap), ptr(proj), ptr(qbuf), ptr(kc), ptr(vc), ptr(norms), ptr(pos), None))
    ffi.check(lib.snl_attend(C.byref(st), C.byref(ap), ptr(proj), ptr(qbuf), ptr(kc), ptr(vc), ptr(want), None, None))
    rope = torch.empty(3000, 32, 2, device="cuda")
    paged.rope_table(rope, 1e7)
    per = proj[:, :2 * heads * 256].view(n, heads, 512)
    q_out = torch.empty(n, heads, 256, dtype=F16, device="cuda")
    p.cache(paged).append(p.batch(paged), per[:, :, :256], proj[:, 2 * heads * 256:(2 * heads + kv) * 256].view(n, kv, 256),
                          proj[:, (2 * heads + kv) * 256:].view(n, kv, 256), q_out, pos, rope, axes=paged.INTERLEAVED,
                          sections=(11, 11, 10), q_norm=norms[:256].contiguous(), k_norm=norms[256:].contiguous())
    pg, sl = p.where(0)
    # the engine's 32-bit angles at positions up to 3000 are off by up to 2e-4
    assert (p.k[pg, :, sl].float() - kc.view(n, kv, 256).float()).abs().max() < 5e-3
    assert torch.equal(p.v[pg, :, sl], vc.view(n, kv, 256))
    out, _ = run_attend(p, q_out, per[:, :, 256:], out_dtype=F32)
    assert (out.view(n, -1) - want).abs().max() < 4e-3 * want.abs().max()


def test_serving_example(lib, capsys):
    """The example's prompts, eviction and tokens; chunks of a prompt give what one chunk does."""
    import sys
    from pathlib import Path

    sys.path.insert(0, str(Path(paged.__file__).resolve().parent.parent / "examples"))
    import paged_serving as ex

    out, layer = ex.serve(budget=192, steps=3)
    assert layer.lens == [195, 48, 132] and layer.seen == [303, 48, 132] and out.isfinite().all()
    assert sorted(layer.free + [p for t in layer.tables for p in t]) == list(range(128))
    again, _ = ex.serve(budget=192, steps=3)
    assert torch.equal(out, again)
    x = torch.randn(200, 256, device="cuda")
    a, b = (ex.PagedLayer(ex.small(), pages=32) for _ in range(2))
    whole = a.step([a.add()], [x])
    s = b.add()
    parts = torch.cat([b.step([s], [x[i:j]]) for i, j in ((0, 150), (150, 151), (151, 200))])
    # values of order 1; the projections' rows come from two kernels (1e-4), attention rounds to 2^-11
    assert (whole - parts).abs().max() < 5e-3 * whole.abs().max()


# A batch for far longer sequences: single rows go by equal shares of all blocks instead of a cluster each.
WIDE = dict(width=20000 // 8, max_len=20000)


@pytest.mark.parametrize("heads,kv,d,page,layout,dtype", [s for s in SHAPES if s[0] // s[1] <= 8])
@pytest.mark.parametrize("lens", [[1], [129], [7, 300, 64, 1], [600, 0, 63, 64, 65, 8, 9] * 3])
def test_attend_one_row_by_equal_shares(heads, kv, d, page, layout, dtype, lens):
    check_attend(Problem(lens, [min(n, 1) for n in lens], heads, kv, d, page, layout, dtype, seed=len(lens), **WIDE))


@pytest.mark.parametrize("mask", MASKS)
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("by_shares", [False, True])
def test_attend_one_row_masks(mask, d, by_shares):
    p = Problem([300, 150, 77, 2000], [1, 1, 1, 1], 8, 2, d, 16, seed=d, **(WIDE if by_shares else {}))
    gate = torch.randn(p.n, p.heads, p.d, device="cuda", generator=torch.Generator("cuda").manual_seed(d))
    check_attend(p, gate=gate, out_dtype=F32, **masks_of(p, **MASKS[mask]))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 7, 9, 18, 37, 75, 150])
@pytest.mark.parametrize("heads,d", [(8, 256), (32, 128)])
def test_attend_one_row_clusters(n, heads, d):
    """Clusters of 8, 4, 2 and 1 CTAs, and more rows than one wave holds."""
    p = Problem([(17 * i) % 480 + 1 for i in range(n)], [1] * n, heads, heads // 4, d, 16, seed=n)
    check_attend(p)
    assert all(torch.equal(a, b) for a, b in zip(run_attend(p), run_attend(p)))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("lens,budget,sink,recent", [
    ([8192, 8191, 700], 300, 4, 32), ([16384, 16389, 4096, 1], 5000, 0, 0), ([33000], 20000, 20000, 0),
    ([40001], 7, 3, 4), ([16400], 16399, 5, 9000),
])
def test_evict_by_clusters(lens, budget, sink, recent, in_place):
    """Lists long enough for 2, 4 or 8 CTAs; few distinct weights, so that equal ones lie in all of them."""
    p = Problem(lens, [min(n, 1) for n in lens], 4, 2, 128, 16, seed=budget, weight=True,
                spare=len(lens) * -(-min(budget, max(lens)) // 16))
    p.weight.copy_((p.weight * 50).floor())
    check_evict(p, budget, sink, recent, in_place)


def test_evict_many_long_lists():
    """More lists than clusters have room for, each of more candidates than one CTA holds keys of."""
    kv, budget, lens = 4, 700, [50001 - 211 * i for i in range(40)]
    p = Problem([50001], [1], kv, kv, 128, 256, seed=41, weight=True, spare=3 * 40)
    p.weight.copy_((p.weight * 4000).floor())
    cache = p.cache(paged)
    lens_t = torch.tensor(lens, dtype=torch.int32, device="cuda")
    start = torch.zeros(41, dtype=torch.int32, device="cuda")
    batch = paged.PagedBatch(p.table.expand(40, -1).contiguous(), start, lens_t, 0, 50001)  # pages that all sequences share
    into = torch.tensor(p.free[:120], dtype=torch.int32, device="cuda").view(40, 3)
    kept, new_lens = torch.empty(40, kv, budget, dtype=torch.int32, device="cuda"), torch.empty_like(lens_t)
    w = p.keys(0, p.weight[..., None])[..., 0].float()  # [slot, kv]
    k, v = p.keys(0, p.k).to(F16), p.keys(0, p.v).to(F16)
    cache.evict(batch, budget, kept, into, new_lens, sink=3, recent=50)
    assert (new_lens == budget).all()
    at = torch.arange(budget, device="cuda")
    for i, n in enumerate(lens):
        order = torch.sort(w[3:n - 50], dim=0, descending=True, stable=True).indices[:budget - 53] + 3
        must = torch.cat([torch.arange(3), torch.arange(n - 50, n)]).cuda()[:, None].expand(-1, kv)
        want = torch.cat([must, order]).sort(0).values.T  # [kv, budget]
        assert torch.equal(kept[i], want.int())
        page = into[i, at // 256].long()
        for h in range(kv):
            for now, was in ((p.k, k), (p.v, v), (p.weight, w)):
                assert torch.equal(now[page, h, at % 256], was[want[h], h])


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("n", [8195, 16384, 40001])
@pytest.mark.parametrize("sink,recent", [(1000, 0), (0, 1000), (100, 4900)])
def test_evict_without_a_choice_by_clusters(n, sink, recent, in_place):
    """A budget of sink and recent slots alone leaves nothing to select: lists of 2, 4 and 8 CTAs."""
    budget = sink + recent
    p = Problem([n, 3000], [1, 1], 2, 2, 128, 16, seed=n, weight=True, spare=2 * -(-budget // 16))
    check_evict(p, budget, sink, recent, in_place)


@pytest.mark.parametrize("n", [8195, 16384, 40001])
def test_evict_without_a_choice_every_time(n):
    p = Problem([n], [1], 2, 2, 128, 16, seed=n, weight=True, spare=200)
    cache, batch, lens = p.cache(paged), p.batch(paged), torch.empty_like(p.len_t)
    into = torch.tensor([p.free[:188]], dtype=torch.int32, device="cuda")
    want = torch.cat([torch.arange(1000), torch.arange(n - 2000, n)]).to(torch.int32).cuda()
    kept = torch.full((100, 1, 2, 3000), 99, dtype=torch.int32, device="cuda")
    for x in kept:
        cache.evict(batch, 3000, x, into, lens, sink=1000, recent=2000)
    assert (kept == want).all()


def test_evict_very_long():
    """More candidates than the shared memory of eight CTAs holds keys of."""
    p = Problem([400000], [1], 1, 1, 128, 256, seed=29, weight=True, spare=20)
    check_evict(p, 5000, 4, 64, False)


@pytest.mark.parametrize("cap", [20.0, 50.0, 1000.0])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("lens,rows", [([3] * 20, [1] * 20), ([9] * 6, [5] * 6), ([40] * 5, [40] * 5)])
def test_attend_far_below_the_cap(lens, rows, d, cap):
    """Scores that the cap hardly changes keep their 32 bits: a score is off by some 2^-22 of itself,
    not of the cap (which at 50 is 1e-5), and so is the log-sum-exp of few keys."""
    p = Problem(lens, rows, 8, 2, d, 16, seed=31, peak=0.3)
    out, lse = run_attend(p, cap=cap)
    _, z, _, _ = ref.attend(p, p.q, None, out_dtype=None, cap=cap)
    s = float(p.q.double().norm(dim=-1).max() * p.k.nan_to_num(0).double().norm(dim=-1).max()) / math.sqrt(d)  # a bound on |s|
    assert ((lse.double() - z).abs() <= 8 * 2.0**-23 * (1 + s + z.abs())).all()


# Kernels of attend: tiles in one part and in several, a row's cluster, equal shares.
EACH_KERNEL = [([300, 150], [37, 50], {}), ([9000], [70], {}), ([300, 150, 77], [1, 1, 1], {}), ([300, 150, 2000], [1, 1, 1], WIDE)]


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("lens,rows,bounds", EACH_KERNEL)
def test_attend_gate_of_rows_without_keys(lens, rows, bounds, d, bad):
    """A padding row is 0 whatever its gate holds."""
    p = Problem(lens, rows, 8, 2, d, seed=d, **bounds)
    off = torch.arange(p.n, device="cuda") % 3 == 1
    first = torch.where(off, 2**31 - 1, 0).to(torch.int32)
    gate = p.normal(p.n, 8, d)
    want, z = run_attend(p, gate=gate, out_dtype=F32, first=first)
    gate[off] = bad
    out, lse = run_attend(p, gate=gate, out_dtype=F32, first=first)
    assert (out[off] == 0).all() and torch.isneginf(lse[off]).all()
    assert torch.equal(out, want) and torch.equal(lse, z)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("lens,rows,bounds", EACH_KERNEL)
def test_attend_gate_of_scores_of_minus_infinity(lens, rows, bounds, d):
    p = Problem(lens, rows, 8, 2, d, seed=d, **bounds)
    p.k[..., 0] = math.inf
    p.q[..., 0] = -1
    out, lse = run_attend(p, gate=torch.full((p.n, 8, d), math.nan, device="cuda"))
    assert (out == 0).all() and torch.isneginf(lse).all()
