"""Paged KV cache: planning a step, rotate-and-append into pages, and attention over pages, against plain numpy
statements in float64 (integers exactly). Each test runs on the CPU oracle and, marked gpu, on the CUDA library; both
compile the same argument checks (csrc/paged_args.h).

Attention tolerance, from u = 2^-24 (half an fp32 step): a score is a dot product of D terms whose operands carry at
most 3·2^-22 = 12u relative error when they are split into two 16-bit parts (the fp32 path has less) plus D roundings,
so it is off by at most (D + 16)·u·A with A = max sum |q||k|·scale; a weight is off by twice that relatively, the sum
over L values adds at most (L + 32)·u, so an output is off by at most max|v|·(2·(D + 16)·A + L + 32)·u. The norm of the
whole error is held to the probabilistic counterpart of that bound (rounding errors of independent sign, factor 8):
8·(2·sqrt(D + 16)·A' + sqrt(L + 32))·u with A' the root mean square of sum |q||k|·scale."""
import numpy as np
import pytest

from projectai_b200 import cabi
from projectai_b200.cabi import ArgumentError, DeviceTimeoutError, InvalidOperationError, OutOfRangeError, UnsupportedError

U = 2.0 ** -24


@pytest.fixture(params=["oracle", pytest.param("cuda", marks=pytest.mark.gpu)])
def be(request):
    return request.getfixturevalue(request.param)


def ceil_div(a, b):
    return -(-a // b)


# ---------------------------------------------------------------- plan
class PlanRef:
    """The plan of pai_paged_plan on host integers."""

    def __init__(self, lengths, new, table, ring, head, count, page, rows):
        self.table, self.ring = table.copy(), ring.copy()
        size, taken, back = len(ring), 0, []
        self.q_start, self.kv_len, self.slots, self.positions = [0], [], [], []
        for i, (length, x) in enumerate(zip(lengths, new)):
            if x < 0:
                back += list(table[i][:ceil_div(length, page)])
            for j in range(ceil_div(length, page), ceil_div(length + x, page) if x > 0 else 0):
                self.table[i][j] = self.ring[(head + taken) % size]
                taken += 1
            for p in range(length, length + max(0, x)):
                self.positions.append(p)
                self.slots.append(self.table[i][p // page] * page + p % page)
            self.q_start.append(self.q_start[-1] + max(0, x))
            self.kv_len.append(length + x if x >= 0 else 0)
        for j, p in enumerate(back):
            self.ring[(head + count + j) % size] = p
        self.slots += [-1] * (rows - len(self.slots))
        self.positions += [0] * (rows - len(self.positions))
        self.state = [(head + taken) % max(1, size), count - taken + len(back)]


def plan_inputs(seed, reqs, page, spare=3, wide=2, head=None):
    """Tables and ring in which the requests hold the pages of their cached tokens, in shuffled order."""
    rng = np.random.default_rng(seed)
    lengths, new = [c for c, _ in reqs], [x for _, x in reqs]
    held = [ceil_div(c, page) for c in lengths]
    need = [ceil_div(c + x, page) - h if x > 0 else 0 for (c, x), h in zip(reqs, held)]
    order = rng.permutation(sum(held) + sum(need) + spare)
    max_pages = max([h + n for h, n in zip(held, need)] + [0]) + wide
    table = np.full((len(reqs), max_pages), -1, np.int64)
    at = 0
    for i, h in enumerate(held):
        table[i, :h] = order[at:at + h]
        at += h
    count = len(order) - at
    head = int(rng.integers(len(order))) if head is None else head
    ring = np.full(len(order), -1, np.int64)
    ring[(head + np.arange(count)) % len(order)] = order[at:]
    return lengths, new, table, ring, head, count


PLANS = [
    ([(0, 1)], 16, 0), ([(15, 1)], 16, 0), ([(16, 1)], 16, 2), ([(5, 0)], 16, 1), ([(5, -1)], 16, 0),
    ([(0, 0), (0, 0)], 4, 3), ([(0, 40), (3, 1), (8, -1), (7, 9), (0, 0), (12, -1)], 4, 5),
    ([(10, 3), (0, 1), (1, 7)], 1, 0), ([(100, 30), (6, 1)], 7, 4), ([(100, 300), (6, 1)], 128, 0), ([], 16, 3), ([], 16, 0),
    ([(i * 7 % 50, (i * 5 % 4) - 1) for i in range(300)], 8, 9),       # more requests than a block has threads
    ([(i % 90, i % 3) for i in range(1000)], 16, 0), ([(33, 2000), (1, 1)], 16, 100),
]


@pytest.mark.parametrize("reqs,page,pad", PLANS)
def test_plan_matches_definition(be, reqs, page, pad):
    lengths, new, table, ring, head, count = plan_inputs(3, reqs, page)
    rows = sum(max(0, x) for x in new) + pad
    ref = PlanRef(lengths, new, table, ring, head, count, page, rows)
    t = [be.from_host(np.array(a, np.float32)) for a in (lengths, new, table, ring, [head, count])]
    for _ in range(2):  # the inputs are not consumed: the same plan again
        got = be.paged_plan(*t, page, rows)
        for name, r in zip(("q_start", "kv_len", "slots", "positions", "state"), got):
            assert be.to_host(r).tolist() == list(map(float, getattr(ref, name))), name
        assert np.array_equal(be.to_host(t[2]), ref.table.astype(np.float32))
        assert np.array_equal(be.to_host(t[3]), ref.ring.astype(np.float32))
    assert be.check_device_error() == 0


def test_plan_reads_strided_operands(be):
    reqs, page = [(9, 4), (3, -1), (0, 6)], 4
    lengths, new, table, ring, head, count = plan_inputs(4, reqs, page, head=2)
    ref = PlanRef(lengths, new, table, ring, head, count, page, 10)
    both = be.from_host(np.array([lengths, new], np.float32).T.copy())  # [N, 2]: columns are strided
    cols = [column(both, i) for i in range(2)]
    wide = be.from_host(np.repeat(table.astype(np.float32), 2, axis=1).copy())
    tv = strided(wide, 1, 2)
    rv = strided(be.from_host(np.repeat(ring.astype(np.float32), 3).copy()), 0, 3)
    sv = strided(be.from_host(np.repeat(np.array([head, count], np.float32), 2).copy()), 0, 2)
    got = be.paged_plan(cols[0], cols[1], tv, rv, sv, page, 10)
    for name, r in zip(("q_start", "kv_len", "slots", "positions", "state"), got):
        assert be.to_host(r).tolist() == list(map(float, getattr(ref, name))), name
    assert np.array_equal(be.to_host(tv), ref.table.astype(np.float32))
    assert np.array_equal(be.to_host(rv), ref.ring.astype(np.float32))
    raw = be.to_host(wide)
    assert np.array_equal(raw[:, 1::2], np.repeat(table, 2, axis=1)[:, 1::2].astype(np.float32))  # between the strides: untouched


def column(t, i):
    r = t.copy_desc()
    r.rank, r.dims[0], r.strides[0], r.offset = 1, t.dims[0], t.strides[0], t.offset + i * t.strides[1]
    return r


def strided(t, axis, step):
    """Every step-th element along an axis."""
    r = t.copy_desc()
    r.dims[axis] = t.dims[axis] // step
    r.strides[axis] = t.strides[axis] * step
    return r


@pytest.mark.parametrize("what", ["short ring", "rows", "max_pages", "nan length", "fraction", "negative length", "new below -1",
                                  "head", "count", "huge"])
def test_plan_refuses_what_it_cannot_place(be, what):
    """Values the device finds wrong: error flag, nothing allocated, no token gets a slot."""
    reqs, page = [(20, 5), (7, 6), (9, -1)], 4
    lengths, new, table, ring, head, count = plan_inputs(5, reqs, page, spare=0, wide=0)
    lengths, new, state, rows = [float(x) for x in lengths], [float(x) for x in new], [float(head), float(count)], 12
    if what == "short ring": state[1] -= 1
    if what == "rows": rows = 10
    if what == "max_pages": new[0], rows = 6.0 + 4 * table.shape[1], 100
    if what == "nan length": lengths[1] = float("nan")
    if what == "fraction": new[1] = 1.5
    if what == "negative length": lengths[0] = -1.0
    if what == "new below -1": new[2] = -2.0
    if what == "head": state[0] = float(len(ring))
    if what == "count": state[1] = float(len(ring) + 1)
    if what == "huge": lengths[0] = 3.0e38
    t = [be.from_host(np.array(a, np.float32)) for a in (lengths, new, table, ring, state)]
    q_start, kv_len, slots, positions, nxt = be.paged_plan(*t, page, rows)
    with pytest.raises(DeviceTimeoutError):
        be.check_device_error()
    assert be.to_host(q_start).tolist() == [0.0] * 4
    assert be.to_host(slots).tolist() == [-1.0] * rows and be.to_host(positions).tolist() == [0.0] * rows
    assert np.array_equal(be.to_host(nxt), np.array(state, np.float32))
    assert np.array_equal(be.to_host(t[2]), table.astype(np.float32)) and np.array_equal(be.to_host(t[3]), ring.astype(np.float32))
    kept = [x if np.isfinite(x) and x >= 0 and x == int(x) and x <= table.shape[1] * page else 0.0 for x in lengths]
    assert be.to_host(kv_len).tolist() == kept


def test_plan_of_wrongly_named_pages(be):
    """A page id outside [0, pages) leaves its tokens without a slot; the others keep theirs."""
    table = np.array([[2, 9], [0, -1]], np.float32)  # request 0's second page does not exist
    t = [be.from_host(np.array(a, np.float32)) for a in ([6, 3], [2, 1], table, [1, 3, 0, 0], [0, 2])]
    _, _, slots, positions, _ = be.paged_plan(*t, 4, 3)
    assert be.to_host(slots).tolist() == [-1.0, -1.0, 3.0] and be.to_host(positions).tolist() == [6.0, 7.0, 3.0]
    with pytest.raises(DeviceTimeoutError):
        be.check_device_error()


def test_plan_refusals(be):
    def call(lengths=(3,), new=(1,), table=((0, 1),), ring=(0, 1, 2), state=(0, 1), page=4, rows=1):
        t = [x if isinstance(x, cabi.PaiTensor) else be.from_host(np.array(x, np.float32)) for x in (lengths, new, table, ring, state)]
        return be.paged_plan(*t, page, rows)

    call()
    for kw in (dict(new=(1, 2)), dict(table=((0, 1), (1, 2))), dict(state=(0, 1, 2)), dict(lengths=((3,),)), dict(ring=((0,),))):
        with pytest.raises(ArgumentError):
            call(**kw)
    for kw in (dict(page=0), dict(page=-3), dict(rows=-1)):
        with pytest.raises(OutOfRangeError):
            call(**kw)
    for kw in (dict(page=1 << 23), dict(rows=(1 << 24) + 1)):
        with pytest.raises(UnsupportedError):
            call(**kw)
    row = be.from_host(np.array([[0, 1]], np.float32))
    with pytest.raises(ArgumentError):
        call(lengths=(3, 3), new=(1, 1), table=cabi.broadcast_to(row, (2, 2)))
    shared = be.from_host(np.array([3.0], np.float32))
    call(lengths=shared, new=shared)  # inputs may be one tensor
    with pytest.raises(ArgumentError):
        call(lengths=shared, ring=shared, state=(0, 0))
    gone, *rest = (be.from_host(np.array(x, np.float32)) for x in ((3,), (1,), ((0, 1),), (0, 1, 2), (0, 1)))
    be.release(gone)  # nothing is allocated from here to the call: the block cannot belong to another tensor again
    with pytest.raises(InvalidOperationError):
        be.paged_plan(gone, *rest, 4, 1)


# ---------------------------------------------------------------- append
def tables(rows, d):
    freq = 10000.0 ** (-np.arange(0, d, 2) / d)
    ang = np.arange(rows)[:, None] * freq
    ang = np.concatenate([ang, ang], 1)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def turned(x, c, s):
    """RotaryEmbedding of float32 rows, each operation rounded once."""
    h = x.shape[-1] // 2
    c, s = c[:, None], s[:, None]
    lo = x[..., :h] * c[..., :h] + -x[..., h:] * s[..., :h]
    hi = x[..., h:] * c[..., h:] + x[..., :h] * s[..., h:]
    return np.concatenate([lo, hi], -1)


def append_ref(q, k, v, cos, sin, pos, slots, kc, vc):
    page = kc.shape[2]
    kc, vc = kc.copy(), vc.copy()
    kr = turned(k, cos[pos], sin[pos])
    for t, s in enumerate(slots):
        if s >= 0:
            kc[s // page, :, s % page] = kr[t]
            vc[s // page, :, s % page] = v[t]
    return turned(q, cos[pos], sin[pos]), kc, vc


def rnd(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


@pytest.mark.parametrize("rows,h,kvh,d,page,pages", [(1, 4, 2, 64, 16, 3), (1, 1, 1, 2, 1, 2), (5, 12, 12, 64, 24, 4), (33, 8, 2, 16, 5, 20),
                                                     (7, 3, 1, 6, 3, 9), (40, 6, 3, 128, 8, 11), (700, 32, 8, 64, 16, 60), (0, 4, 2, 64, 16, 3),
                                                     (9, 2, 2, 20, 4, 5), (3, 2, 1, 200, 4, 2)])
def test_append_matches_rounded_definition(be, rows, h, kvh, d, page, pages):
    rng = np.random.default_rng(rows)
    slots = rng.permutation(pages * page)[:rows].astype(np.int64)
    if rows > 2:
        slots[rng.integers(rows)] = -1
    pos = rng.integers(0, 50, rows)
    cos, sin = tables(50, d)
    q, k, v, kc, vc = rnd(1, rows, h, d), rnd(2, rows, kvh, d), rnd(3, rows, kvh, d), rnd(4, pages, kvh, page, d), rnd(5, pages, kvh, page, d)
    ref = append_ref(q, k, v, cos, sin, pos, slots, kc, vc)
    tkc, tvc = be.from_host(kc), be.from_host(vc)
    out = be.paged_rope_append(*map(be.from_host, (q, k, v, cos, sin)), be.from_host(pos), be.from_host(slots), tkc, tvc)
    for name, want, got in zip(("q", "k_cache", "v_cache"), ref, (out, tkc, tvc)):
        assert np.array_equal(want, be.to_host(got)), name
    assert be.check_device_error() == 0


@pytest.mark.parametrize("shift", [0, 1])
def test_append_of_strided_views(be, shift):
    """q, k and v as views of one product, caches as views with room between heads and positions in another order;
    shift moves the rows off 16-byte boundaries."""
    rows, h, kvh, d, page, pages = 6, 4, 2, 16, 4, 5
    x = rnd(7, rows, (h + 2 * kvh) * d + shift)
    whole = cabi.slice_view(be.from_host(x), 1, shift, (h + 2 * kvh) * d)
    parts = []
    for at, n in ((0, h), (h, kvh), (h + kvh, kvh)):
        r = whole.copy_desc()
        r.rank, r.offset = 3, whole.offset + at * d
        for i, (n_, s_) in enumerate(((rows, whole.strides[0]), (n, d), (d, 1))):
            r.dims[i], r.strides[i] = n_, s_
        parts.append(r)
    q, k, v = (be.to_host(t) for t in parts)
    raw = rnd(8, 2, pages, page, kvh + 1, d + shift)
    store = be.from_host(raw)
    caches = []
    for i in range(2):
        r = store.copy_desc()  # [pages, kvh, page, d] over storage [2, pages, page, kvh + 1, d + shift]
        r.rank, r.offset = 4, i * store.strides[0] + shift
        for a, (n_, s_) in enumerate(((pages, store.strides[1]), (kvh, store.strides[3]), (page, store.strides[2]), (d, 1))):
            r.dims[a], r.strides[a] = n_, s_
        caches.append(r)
    cos, sin = tables(9, d)
    pos, slots = np.array([0, 8, 3, 3, 1, 2]), np.array([19, 0, 7, -1, 4, 11])
    ref = append_ref(q, k, v, cos, sin, pos, slots, be.to_host(caches[0]), be.to_host(caches[1]))
    out = be.paged_rope_append(*parts, *map(be.from_host, (cos, sin, pos, slots)), *caches)
    for want, got in zip(ref, (out, *caches)):
        assert np.array_equal(want, be.to_host(got))
    after = be.to_host(store)
    assert np.array_equal(after[..., kvh, :], raw[..., kvh, :])  # what lies between the views is untouched
    assert be.check_device_error() == 0


@pytest.mark.parametrize("pos,slot", [([0, 1, 2], [3, 99, 4]), ([0, 50, 2], [3, 1, 4]), ([0, 1, 2], [3, 1.5, 4]), ([0, float("nan"), 2], [3, 1, 4]),
                                      ([0, -1, 2], [3, 1, 4]), ([0, 1, 2], [3, -2, 4]), ([0, 1, 2], [3, float("inf"), 4])])
def test_append_skips_wrong_slots_and_positions(be, pos, slot):
    d, page, pages = 16, 4, 2
    cos, sin = tables(50, d)
    q, k, v, kc, vc = rnd(1, 3, 2, d), rnd(2, 3, 1, d), rnd(3, 3, 1, d), rnd(4, pages, 1, page, d), rnd(5, pages, 1, page, d)
    keep = [0, 2]
    ref = append_ref(q[keep], k[keep], v[keep], cos, sin, np.array(pos)[keep].astype(int), np.array(slot)[keep].astype(int), kc, vc)
    tkc, tvc = be.from_host(kc), be.from_host(vc)
    out = be.to_host(be.paged_rope_append(*map(be.from_host, (q, k, v, cos, sin, pos, slot)), tkc, tvc))
    with pytest.raises(DeviceTimeoutError):
        be.check_device_error()
    assert np.array_equal(out[keep], ref[0])
    assert np.array_equal(be.to_host(tkc), ref[1]) and np.array_equal(be.to_host(tvc), ref[2])
    if pos[1] != 1:
        assert not out[1].any()


def test_append_refusals(be):
    d, page = 16, 4
    cos, sin = tables(8, d)
    base = dict(q=rnd(1, 3, 4, d), k=rnd(2, 3, 2, d), v=rnd(3, 3, 2, d), cos=cos, sin=sin, pos=[0, 1, 2], slots=[0, 1, 2],
                kc=rnd(4, 5, 2, page, d), vc=rnd(5, 5, 2, page, d))

    def call(**kw):
        t = [x if isinstance(x, cabi.PaiTensor) else be.from_host(np.asarray(x, np.float32)) for x in (base | kw).values()]
        return be.paged_rope_append(*t)

    call()
    for kw in (dict(v=rnd(3, 3, 1, d)), dict(pos=[0, 1]), dict(slots=[0, 1, 2, 3]), dict(k=rnd(2, 4, 2, d), v=rnd(2, 4, 2, d)),
               dict(kc=rnd(4, 5, 1, page, d), vc=rnd(4, 5, 1, page, d)), dict(vc=rnd(4, 6, 2, page, d)), dict(cos=cos[:, :8]),
               dict(q=rnd(1, 3, 4, 8)), dict(q=rnd(1, 3, d)), dict(kc=rnd(4, 5, page, d)), dict(sin=sin[:4])):
        with pytest.raises(ArgumentError):
            call(**kw)
    odd = dict(q=rnd(1, 3, 4, 15), k=rnd(2, 3, 2, 15), v=rnd(3, 3, 2, 15), cos=cos[:, :15], sin=sin[:, :15], kc=rnd(4, 5, 2, page, 15),
               vc=rnd(5, 5, 2, page, 15))
    with pytest.raises(ArgumentError):
        call(**odd)
    one = be.from_host(base["kc"])
    with pytest.raises(ArgumentError):
        call(kc=one, vc=one)
    flat = be.from_host(rnd(6, 1, 2, page, d))
    with pytest.raises(ArgumentError):
        call(kc=cabi.broadcast_to(flat, (5, 2, page, d)), vc=cabi.broadcast_to(be.from_host(rnd(7, 1, 2, page, d)), (5, 2, page, d)))
    with pytest.raises(UnsupportedError):
        call(q=cabi.transpose(be.from_host(rnd(1, 3, d, 4)), 1, 2))


def test_append_refuses_tables_whose_rows_f32_cannot_name(be):
    """Beyond 2^24 rows the largest position rounds up to one behind the table: 2^24 + 4 rows, position 2^24 + 4."""
    d, rows = 16, (1 << 24) + 4
    kc, vc = be.from_host(rnd(4, 2, 1, 4, d)), be.from_host(rnd(5, 2, 1, 4, d))
    args = [be.from_host(rnd(s, 1, n, d)) for s, n in ((1, 2), (2, 1), (3, 1))]
    one = be.from_host(rnd(6, 1, d))
    for n in (rows, 1 << 24):
        wide = cabi.broadcast_to(one, (n, d))
        call = lambda: be.paged_rope_append(*args, wide, wide, be.from_host([(1 << 24) - 1.0]), be.from_host([1.0]), kc, vc)  # noqa: E731
        if n > 1 << 24:
            with pytest.raises(UnsupportedError):
                call()
        else:
            call()
    assert be.check_device_error() == 0


def view(t, offset, dims, strides):
    r = t.copy_desc()
    r.rank, r.offset = len(dims), offset
    for i, (n, s) in enumerate(zip(dims, strides)):
        r.dims[i], r.strides[i] = n, s
    return r


def test_plan_refuses_operands_that_share_elements(be):
    """One buffer of [N, 2 + max_pages + ...]: columns of their own are fine, shared ones are not."""
    n, pages = 3, 4
    big = be.from_host(np.zeros(200, np.float32))
    packed = [view(big, 0, (n,), (6,)), view(big, 1, (n,), (6,)), view(big, 2, (n, pages), (6, 1)), view(big, 100, (9,), (2,)), view(big, 101, (2,), (2,))]
    be.paged_plan(*packed, 4, 2)  # lengths, new_tokens and table interleaved, ring and state too
    assert be.check_device_error() == 0
    for i, wrong in ((0, view(big, 2, (n,), (6,))), (1, view(big, 5, (n,), (6,))), (1, view(big, 17, (n,), (-6,))), (2, view(big, 98, (n, pages), (6, 1))),
                     (3, view(big, 13, (9,), (1,))), (4, view(big, 100, (2,), (2,))), (4, view(big, 102, (2,), (1,)))):
        args = list(packed)
        args[i] = wrong
        with pytest.raises(ArgumentError):
            be.paged_plan(*args, 4, 2)


def test_append_refuses_caches_that_share_elements(be):
    d, page, pages, kvh = 16, 4, 5, 2
    cos, sin = tables(8, d)
    both = be.from_host(np.zeros((pages, 2, kvh, page, d), np.float32))  # keys and values of a page side by side
    step, at = (2 * kvh * page * d, page * d, d, 1), kvh * page * d
    kc, vc = view(both, 0, (pages, kvh, page, d), step), view(both, at, (pages, kvh, page, d), step)
    q, k, v = be.from_host(rnd(1, 3, 4, d)), be.from_host(rnd(2, 3, kvh, d)), be.from_host(rnd(3, 3, kvh, d))
    rest = [be.from_host(np.asarray(x, np.float32)) for x in (cos, sin, [0, 1, 2], [0, 1, 2])]
    be.paged_rope_append(q, k, v, *rest, kc, vc)
    assert be.check_device_error() == 0
    for a, b in ((kc, view(both, at - d, (pages, kvh, page, d), step)), (kc, view(both, 2 * at, (pages - 1, kvh, page, d), step)),
                 (view(both, 8, (pages - 1, kvh, page, d), step), vc)):
        p = min(a.dims[0], b.dims[0])
        with pytest.raises(ArgumentError):
            be.paged_rope_append(q, k, v, *rest, *(view(x, x.offset, (p, kvh, page, d), step) for x in (a, b)))
    inside = view(both, at, (3, kvh, d), (page * d, d, 1))  # rows of the value cache
    for args in ((q, inside, v), (q, k, inside), (view(both, 0, (3, 4, d), (4 * d, d, 1)), k, v)):
        with pytest.raises(ArgumentError):
            be.paged_rope_append(*args, *rest, kc, vc)
    for i in range(4):
        wrong = list(rest)
        wrong[i] = view(both, 3, tuple(rest[i].dims[:rest[i].rank]), tuple(rest[i].strides[:rest[i].rank]))
        with pytest.raises(ArgumentError):
            be.paged_rope_append(q, k, v, *wrong, kc, vc)


# ---------------------------------------------------------------- attention
def attend_ref(q, kc, vc, table, q_start, kv_len, scale):
    """float64, row by row; also max and root mean square of sum |q||k| scale for the tolerance."""
    rows, h, d = q.shape
    page, g = kc.shape[2], h // kc.shape[1]
    out = np.zeros((rows, h, d))
    most, squares, count = 0.0, 0.0, 0
    for i in range(len(kv_len)):
        a, b, length = q_start[i], q_start[i + 1], kv_len[i]
        ids = table[i, :ceil_div(length, page)]
        k = kc[ids].transpose(1, 0, 2, 3).reshape(kc.shape[1], -1, d)[:, :length].astype(np.float64)
        v = vc[ids].transpose(1, 0, 2, 3).reshape(kc.shape[1], -1, d)[:, :length].astype(np.float64)
        for r in range(a, b):
            p = length - (b - a) + (r - a)
            if p < 0:
                continue
            for j in range(h):
                kk, x = k[j // g, :p + 1], q[r, j].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    s = kk @ x * scale
                    w = np.exp(s - s.max())
                    out[r, j] = w @ v[j // g, :p + 1] / w.sum()
                    size = np.abs(kk) @ np.abs(x) * scale
                if np.isfinite(size).all():
                    most, squares, count = max(most, size.max()), squares + float(size @ size), count + size.size
    return out, most, np.sqrt(squares / max(1, count))


def check_attention(ref, got, d, longest, vmax, most, rms, scale_of=None):
    err = np.abs(ref - got)
    tol = vmax * (2 * (d + 16) * most + longest + 32) * U
    assert np.isfinite(got).all()
    assert err.max(initial=0.0) <= tol, f"max error {err.max():.3e} > {tol:.3e}"
    norm = np.linalg.norm(ref)
    if norm > 0:
        rel, lim = np.linalg.norm(ref - got) / norm, 8 * (2 * np.sqrt(d + 16) * rms + np.sqrt(longest + 32)) * U
        assert rel <= lim, f"error of the norm {rel:.3e} > {lim:.3e}"


def paged_case(seed, h, kvh, d, page, reqs, pad=0, stale=np.nan):
    """Caches whose unattended positions hold `stale`, table, q_start, kv_len; reqs are (cached, new)."""
    rng = np.random.default_rng(seed)
    total = [c + x for c, x in reqs]
    held = [ceil_div(t, page) for t in total]
    pages = sum(held) + 2
    order = rng.permutation(pages)
    table = np.full((len(reqs), max(held + [0]) + 1), -1, np.int64)
    kc, vc = np.full((pages, kvh, page, d), stale, np.float32), np.full((pages, kvh, page, d), stale, np.float32)
    at = 0
    for i, (n, t) in enumerate(zip(held, total)):
        table[i, :n] = order[at:at + n]
        at += n
        for j in range(t):
            kc[table[i, j // page], :, j % page] = rng.standard_normal((kvh, d))
            vc[table[i, j // page], :, j % page] = rng.standard_normal((kvh, d))
    q_start = np.concatenate([[0], np.cumsum([x for _, x in reqs])]).astype(np.int64)
    q = rng.standard_normal((int(q_start[-1]) + pad, h, d)).astype(np.float32)
    return q, kc, vc, table, q_start, np.array(total, np.int64)


def dirty(be, shape):
    """Fills what the allocator hands out next for this shape with NaN."""
    t = be.from_host(np.full(shape, np.nan, np.float32))
    be.release(t)


def attend(be, q, kc, vc, table, q_start, kv_len, scale, max_new=0):
    dirty(be, q.shape)
    return be.to_host(be.sdpa_paged(*[x if isinstance(x, cabi.PaiTensor) else be.from_host(x) for x in (q, kc, vc, table, q_start, kv_len)], scale, max_new))


ATTEND = [
    (4, 2, 64, 16, [(0, 1)], 0), (12, 12, 64, 16, [(517, 1)], 0), (32, 8, 64, 16, [(100, 1), (0, 1), (31, 1), (700, 1)], 0),
    (8, 2, 16, 5, [(7, 3), (0, 5), (64, 1)], 2), (4, 1, 64, 16, [(63, 2), (62, 2), (64, 2)], 0), (8, 1, 32, 8, [(130, 1)], 1),
    (2, 2, 128, 16, [(200, 3)], 0), (3, 1, 20, 7, [(50, 2), (0, 0), (3, 1)], 0), (2, 1, 6, 3, [(10, 4)], 0), (1, 1, 1, 1, [(5, 1)], 0),
    (16, 1, 64, 16, [(255, 1), (256, 1)], 0),                                                    # 16 rows of one kv head
    (4, 2, 64, 16, [(0, 130)], 0), (8, 2, 64, 16, [(300, 257), (5, 1), (0, 0), (77, 64)], 5), (12, 12, 64, 24, [(301, 60)], 0),
    (8, 2, 16, 5, [(3, 200), (1, 1)], 1), (4, 4, 64, 1, [(40, 33)], 0), (2, 1, 48, 128, [(500, 90)], 0), (6, 2, 64, 64, [(127, 1), (0, 128), (1, 127)], 0),
    (2, 1, 100, 16, [(70, 40)], 0), (2, 2, 7, 4, [(30, 20)], 3), (2, 1, 64, 16, [], 4), (8, 2, 64, 16, [(0, 0)], 3),
    (32, 8, 64, 16, [(120, 6), (1, 6), (500, 3)], 0),
]


@pytest.mark.parametrize("h,kvh,d,page,reqs,pad", ATTEND)
def test_attention_matches_float64(be, h, kvh, d, page, reqs, pad):
    case = paged_case(11, h, kvh, d, page, reqs, pad)
    scale = 1.0 / np.sqrt(d)
    ref, most, rms = attend_ref(*case, scale)
    longest = max([c + x for c, x in reqs] + [0])
    vmax = np.nanmax(np.abs(case[2]), initial=0.0)
    tight = max([x for _, x in reqs] + [1])
    for max_new in (0, tight):
        got = attend(be, *case, scale, max_new)
        check_attention(ref, got, d, longest, vmax, most, rms)
    assert be.check_device_error() == 0


@pytest.mark.parametrize("h,kvh,d,page,reqs", [(32, 8, 64, 16, [(1500, 1), (3, 300), (40, 1), (900, 129), (2047, 1)]), (12, 12, 64, 16, [(1700, 5), (33, 64)]),
                                               (4, 1, 64, 64, [(9000, 1), (20000, 7)]), (2, 2, 64, 16, [(60, 900)])])
@pytest.mark.gpu
def test_attention_of_long_and_mixed_requests(cuda, h, kvh, d, page, reqs):
    case = paged_case(13, h, kvh, d, page, reqs, 3)
    ref, most, rms = attend_ref(*case, 0.125)
    got = attend(cuda, *case, 0.125, max(x for _, x in reqs))
    check_attention(ref, got, d, max(c + x for c, x in reqs), np.nanmax(np.abs(case[2])), most, rms)
    again = attend(cuda, *case, 0.125, max(x for _, x in reqs))
    assert np.array_equal(got, again)  # split work is joined in one order
    assert cuda.check_device_error() == 0


@pytest.mark.parametrize("new", [1, 3, 70])
def test_attention_of_many_requests(be, new):
    """More requests than a block has threads."""
    reqs = [(i % 37, new if i % 5 == 0 else 1) for i in range(300)]
    case = paged_case(17, 2, 1, 16, 8, reqs)
    ref, most, rms = attend_ref(*case, 0.25)
    check_attention(ref, attend(be, *case, 0.25, new), 16, 110, np.nanmax(np.abs(case[2])), most, rms)
    assert be.check_device_error() == 0


@pytest.mark.parametrize("h,new", [(16, 1), (16, 2), (32, 2), (64, 2), (64, 6)])
@pytest.mark.gpu
def test_attention_of_more_requests_than_a_block_lists(cuda, h, new):
    """900 requests of 16 kv heads and a few keys: each block's share is more (request, kv head) pairs than it lists at a
    time, and some of its requests are empty."""
    reqs = [((i * 7) % 11, 0 if i % 9 == 4 else 1 + i % new) for i in range(900)]
    case = paged_case(61, h, 16, 16, 4, reqs, 1)
    ref, most, rms = attend_ref(*case, 0.25)
    check_attention(ref, attend(cuda, *case, 0.25, new), 16, 16, np.nanmax(np.abs(case[2])), most, rms)
    assert cuda.check_device_error() == 0


@pytest.mark.gpu
def test_attention_of_a_table_of_very_many_positions(cuda):
    """8192 requests of up to 2^24 positions (one page, over and over), a few of them with keys."""
    n, h, kvh, d, page = 1 << 13, 4, 2, 16, 4
    new, length = np.zeros(n, np.int64), np.zeros(n, np.int64)
    for i, (x, t) in {0: (1, 700), 5: (2, 300), 4000: (1, 256), 4001: (1, 257), n - 1: (2, 1000)}.items():
        new[i], length[i] = x, t
    rng = np.random.default_rng(79)
    kc, vc = (rng.standard_normal((1, kvh, page, d)).astype(np.float32) for _ in range(2))
    q_start = np.concatenate([[0], np.cumsum(new)])
    q = rng.standard_normal((int(q_start[-1]), h, d)).astype(np.float32)
    ref, most, rms = attend_ref(q, kc, vc, np.zeros((n, 250), np.int64), q_start, length, 0.25)
    table = cabi.broadcast_to(cuda.from_host(np.zeros((1, 1), np.float32)), (n, (1 << 24) // page))
    check_attention(ref, attend(cuda, q, kc, vc, table, q_start, length, 0.25, 2), d, 1000, np.abs(vc).max(), most, rms)
    assert cuda.check_device_error() == 0


@pytest.mark.gpu
def test_two_captured_calls_and_eager_ones_share_the_context(cuda):
    """A captured decode step of split requests and a captured chunk, replayed in turn with eager calls between them."""
    cases = [paged_case(67, 8, 2, 64, 16, [(3000, 1), (9, 1)]), paged_case(71, 8, 2, 64, 16, [(1200, 90), (700, 1)]),
             paged_case(73, 8, 2, 64, 16, [(2000, 2)])]
    refs = [attend_ref(*c, 0.125) for c in cases]
    held = [[cuda.from_host(x) for x in c] for c in cases]
    new = [1, 90, 2]
    graphs = []
    for i in range(2):
        cuda.sdpa_paged(*held[i], 0.125, new[i])
        cuda.graph_begin()
        out = cuda.sdpa_paged(*held[i], 0.125, new[i])
        graphs.append((cuda.graph_end(), out))

    def check(i, got):
        ref, most, rms = refs[i]
        check_attention(ref, got, 64, 3001, np.nanmax(np.abs(cases[i][2])), most, rms)

    for i in (0, 1, 1, 0, 1, 0):
        graph, out = graphs[i]
        cuda.graph_launch(graph)
        eager = cuda.sdpa_paged(*held[2], 0.125, 2)
        check(i, cuda.to_host(out))
        check(2, cuda.to_host(eager))
        cuda.release(eager)
    assert cuda.check_device_error() == 0
    for graph, _ in graphs:
        cuda.graph_destroy(graph)


@pytest.mark.gpu
def test_a_context_can_be_created_while_another_captures(cuda, cuda_lib):
    case = paged_case(131, 8, 2, 64, 16, [(300, 1), (9, 1)])
    held = [cuda.from_host(x) for x in case]
    ref, most, rms = attend_ref(*case, 0.125)
    cuda.sdpa_paged(*held, 0.125, 1)
    cuda.graph_begin()
    out = cuda.sdpa_paged(*held, 0.125, 1)
    other = cabi.NativeBackend(cuda_lib, 0)
    graph = cuda.graph_end()
    cuda.graph_launch(graph)
    check_attention(ref, cuda.to_host(out), 64, 301, np.nanmax(np.abs(case[2])), most, rms)
    check_attention(ref, attend(other, *case, 0.125, 1), 64, 301, np.nanmax(np.abs(case[2])), most, rms)
    assert cuda.check_device_error() == 0 and other.check_device_error() == 0
    cuda.graph_destroy(graph)
    other.close()


@pytest.mark.parametrize("new", [2, 90])
def test_rows_without_keys_and_rows_of_no_request_are_zero(be, new):
    q, kc, vc, table, q_start, kv_len = paged_case(19, 4, 2, 64, 16, [(0, new), (5, 1)], 2)
    kv_len = kv_len.copy()
    kv_len[0] = new - 1  # its first row stands at position -1
    q_start = np.append(q_start, q_start[-1])
    table, kv_len = np.append(table, [[0] * table.shape[1]], 0), np.append(kv_len, 0)
    ref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.125)
    got = attend(be, q, kc, vc, table, q_start, kv_len, 0.125, new)
    assert not got[0].any() and not got[new + 1:].any() and got[1:new + 1].any()
    check_attention(ref, got, 64, new + 5, np.nanmax(np.abs(vc)), most, rms)
    got = attend(be, q, kc, vc, table, q_start + 1, kv_len, 0.125, new)  # the first row belongs to nobody now
    assert not got[0].any()
    assert be.check_device_error() == 0


@pytest.mark.parametrize("reqs,max_new", [([(9, 3)], 3), ([(200, 70), (3, 1)], 70), ([(40, 130)], 0)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_positions_a_row_does_not_attend_may_hold_anything(be, reqs, max_new, bad):
    """The last new token's key and value are not finite: only the last row sees them."""
    q, kc, vc, table, q_start, kv_len = paged_case(23, 4, 2, 64, 16, reqs, 0, stale=bad)
    j = int(kv_len[0]) - 1
    last = int(q_start[1]) - 1
    ref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.125)
    clean_v = np.abs(vc[np.isfinite(vc)]).max()
    vc[table[0, j // 16], 0, j % 16, 5] = bad
    got = attend(be, q, kc, vc, table, q_start, kv_len, 0.125, max_new)
    assert not np.isfinite(got[last, :2, 5]).any()
    fine = np.ones(got.shape, bool)
    fine[last, :2, 5] = False
    check_attention(np.where(fine, ref, 0), np.where(fine, got, 0), 64, int(kv_len.max()), clean_v, most, rms)
    kc[table[0, j // 16], :, j % 16] = bad
    got = attend(be, q, kc, vc, table, q_start, kv_len, 0.125, max_new)
    rest = np.arange(len(q)) != last
    check_attention(ref[rest], got[rest], 64, int(kv_len.max()), clean_v, most, rms)


@pytest.mark.parametrize("reqs", [[(40, 1), (3, 1)], [(70, 100)]])
@pytest.mark.parametrize("size", [1e-12, 1e-3, 3e4, 1e12])
def test_attention_of_large_and_small_values(be, reqs, size):
    """Values far from 1 lose nothing: v scales the result, and q down as k up leaves the scores."""
    q, kc, vc, table, q_start, kv_len = paged_case(29, 4, 2, 64, 16, reqs, 0, stale=0.0)
    size = np.float32(2.0 ** np.round(np.log2(size)))  # a power of two, exact in every product
    ref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.125)
    vmax = np.abs(vc).max()
    got = attend(be, q / size, kc * size, vc * size, table, q_start, kv_len, 0.125)
    check_attention(ref, got / np.float64(size), 64, 170, vmax, most, rms)


@pytest.mark.parametrize("reqs", [[(40, 1), (3, 1)], [(70, 100)]])
def test_attention_of_a_few_large_keys_among_small_ones(be, reqs):
    """One key far above the others in its neighbourhood: the small keys' scores keep their precision."""
    q, kc, vc, table, q_start, kv_len = paged_case(31, 4, 2, 64, 16, reqs, 0, stale=0.0)
    kc *= np.float32(0.05)
    kc[table[0, 1], :, 3] *= np.float32(400.0)
    vc[table[0, 1], :, 5] *= np.float32(1000.0)
    ref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.125)
    got = attend(be, q, kc, vc, table, q_start, kv_len, 0.125)
    check_attention(ref, got, 64, 170, np.abs(vc).max(), most, rms)


def fours(x):
    """Each number replaced by the largest of its group of four adjacent ones."""
    g = np.abs(x.astype(np.float64)).reshape(*x.shape[:-1], -1, 4).max(-1, keepdims=True)
    return np.broadcast_to(g, (*g.shape[:-1], 4)).reshape(x.shape)


def attend_bound(q, kc, vc, table, q_start, kv_len, scale, size=np.abs):
    """float64 result and a bound of its error for each element. With w_j the weights of the row, a score's error is at
    most (D + 16) u sum |q||k| scale (see above), which bends its weight by twice that, e_j, relatively, and the sums add
    (L + 32) u: |error of o_d| <= sum_j w_j |v_jd| (e_j + (L + 32) u) + |o_d| sum_j w_j e_j. Keys of weight 0 count
    for nothing, however large, and so does what other rows attend. A weight is not asked to be exact under 2^-100,
    and its products not under fp32's smallest normal number. `size` is what counts for |x|: abs, or fours."""
    rows, h, d = q.shape
    page, g = kc.shape[2], h // kc.shape[1]
    out, tol = np.zeros((rows, h, d)), np.full((rows, h, d), 2.0 ** -126)  # rows of no request are 0
    for i in range(len(kv_len)):
        a, b, length = q_start[i], q_start[i + 1], kv_len[i]
        ids = table[i, :ceil_div(length, page)]
        k = kc[ids].transpose(1, 0, 2, 3).reshape(kc.shape[1], -1, d)[:, :length].astype(np.float64)
        v = vc[ids].transpose(1, 0, 2, 3).reshape(kc.shape[1], -1, d)[:, :length].astype(np.float64)
        for r in range(a, b):
            n = length - (b - a) + (r - a) + 1
            for j in range(h):
                kk, vv, x = k[j // g, :n], v[j // g, :n], q[r, j].astype(np.float64)
                s = kk @ x * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                e = 2 * (d + 16) * U * (size(kk) @ size(x)) * scale
                out[r, j] = w @ vv
                tol[r, j] = (w * (e + (n + 32) * U) + 2.0 ** -100) @ size(vv) + np.abs(out[r, j]) * (w @ e) + 2.0 ** -126
    return out, tol


def check_bound(be, case, scale, max_new=0, size=np.abs):
    ref, tol = attend_bound(*case, scale, size)
    got = attend(be, *case, scale, max_new).astype(np.float64)
    assert np.isfinite(got).all()
    worst = (np.abs(got - ref) / tol).max()
    assert worst <= 1, f"error {worst:.3g} times its bound"
    assert be.check_device_error() == 0


WIDE = [([(9, 3)], 3, 64), ([(200, 70), (3, 1)], 70, 64), ([(40, 130)], 0, 64), ([(250, 24), (140, 24)], 24, 16)]


def at_key(case, i, j):
    """Page and offset of a request's position."""
    page = case[1].shape[2]
    return case[3][i, j // page], j % page


@pytest.mark.parametrize("reqs,max_new,d", WIDE)
@pytest.mark.parametrize("size", [1e6, 1e8, 1e12, 1e30, 3e38])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_large_number_that_a_row_does_not_attend_changes_nothing(be, reqs, max_new, d, size, which):
    """One element of the last new token's key or value is large: the rows before it do not attend it."""
    case = paged_case(89, 4, 2, d, 16, reqs, 0, stale=0.0)
    p, o = at_key(case, 0, int(case[5][0]) - 1)
    case[1 if which == "k" else 2][p, :, o, 5] = np.float32(size)
    check_bound(be, case, d ** -0.5, max_new)


@pytest.mark.parametrize("reqs,max_new,d", WIDE)
@pytest.mark.parametrize("size", [1e3, 1e6, 1e12, 1e30])
def test_large_keys_of_weight_zero_leave_the_other_scores(be, reqs, max_new, d, size):
    """Keys far below the others in score: attended by every row, weight 0."""
    case = paged_case(97, 4, 2, d, 16, reqs, 0, stale=0.0)
    case[0][..., 5] = np.abs(case[0][..., 5]) + 0.5
    for j in (1, 7):
        p, o = at_key(case, 0, j)
        case[1][p, :, o, 5] = np.float32(-size)
    check_bound(be, case, d ** -0.5, max_new)


@pytest.mark.parametrize("reqs,max_new,d", WIDE)
@pytest.mark.parametrize("size,score", [(1e3, -3.0), (1e6, -12.0), (1e12, -25.0), (1e20, -30.0), (1e30, -60.0), (3e38, -60.0)])
def test_large_values_of_small_weight(be, reqs, max_new, d, size, score):
    """A value that its weight brings down to the size of the others, or above: the weight keeps its precision."""
    case = paged_case(101, 4, 2, d, 16, reqs, 0, stale=0.0)
    case[0][..., 5] = 1.0
    p, o = at_key(case, 0, 3)
    case[1][p, :, o, 5] = np.float32(score * d ** 0.5)
    case[2][p, :, o] *= np.float32(size) / np.abs(case[2][p, :, o]).max()
    check_bound(be, case, d ** -0.5, max_new)


@pytest.mark.parametrize("size,score", [(1e4, -12.0), (1e10, -25.0), (1e16, -30.0), (1e30, -60.0), (1e-10, 20.0), (1e-30, 60.0)])
@pytest.mark.parametrize("reqs,max_new,d", [([(380, 70)], 70, 64), ([(300, 3)], 3, 64), ([(270, 200), (300, 1)], 0, 16)])
def test_stretches_of_large_values_of_small_weight(be, reqs, max_new, d, size, score):
    """Positions 100 to 300 hold values of another size than the rest and scores as far the other way."""
    case = paged_case(103, 4, 2, d, 16, reqs, 0, stale=0.0)
    case[0][..., 5] = 1.0
    for j in range(100, 300):
        p, o = at_key(case, 0, j)
        case[1][p, :, o, 5] = np.float32(score * d ** 0.5)
        case[2][p, :, o] *= np.float32(size)
    check_bound(be, case, d ** -0.5, max_new)


@pytest.mark.parametrize("reqs,max_new,d", WIDE)
@pytest.mark.parametrize("size", [1e7, 1e10, 1e30])
@pytest.mark.parametrize("j", [128, 160])
def test_large_values_in_front_of_a_stretch_that_ends_inside_a_tile(be, reqs, max_new, d, size, j):
    """The first position of 32, with positions that do not exist behind it in the same 32."""
    case = paged_case(109, 4, 2, d, 16, reqs, 0)
    for i in range(len(reqs)):
        if j < case[5][i]:
            p, o = at_key(case, i, j)
            case[2][p, :, o, 5] = np.float32(size)
            case[1][p, :, o, 6] = np.float32(-size)
    check_bound(be, case, d ** -0.5, max_new)


@pytest.mark.parametrize("reqs,max_new,d", WIDE)
@pytest.mark.parametrize("size", [1e5, 1e7, 1e9, 1e11, 1e14, 1e20])
def test_scores_of_any_size(be, reqs, max_new, d, size):
    """Scores whose steps in fp32 are whole powers of two: the largest keeps its weight, with a large value in the tile as well."""
    for big in (False, True):
        q, kc, vc, *rest = paged_case(113, 4, 2, d, 16, reqs, 0, stale=0.0)
        case = [q * np.float32(size), kc, vc, *rest]
        if big:
            p, o = at_key(case, 0, 3)
            vc[p, :, o, 5] = 1e7
        got = attend(be, *case, d ** -0.5, max_new).astype(np.float64)
        assert np.isfinite(got).all()
        ref, tol = attend_bound(*case, d ** -0.5)
        # scores this large are off by more than 1: all a row must do is stay within the values it attends, and follow a key that
        # leads by more than the error
        h = q.shape[1] // kc.shape[1]
        for r in range(len(q)):
            i = int(np.searchsorted(rest[1], r, "right")) - 1
            n = int(rest[2][i] - (rest[1][i + 1] - rest[1][i]) + r - rest[1][i]) + 1
            at = np.arange(n)
            for j in range(q.shape[1]):
                k = kc[rest[0][i, at // 16], j // h, at % 16].astype(np.float64)
                v = vc[rest[0][i, at // 16], j // h, at % 16].astype(np.float64)
                s = k @ case[0][r, j].astype(np.float64) * d ** -0.5
                off = 2 * (d + 16) * U * (np.abs(k) @ np.abs(case[0][r, j]).astype(np.float64)).max() * d ** -0.5
                near = s > s.max() - 2 * off - 100  # beyond that, less than 2^-100
                lo, hi = v[near].min(0), v[near].max(0)
                slack = (n + 32) * U * np.abs(v[near]).max(0) + 2.0 ** -90 * np.abs(v).max(0)
                assert (got[r, j] >= lo - slack).all() and (got[r, j] <= hi + slack).all()
        assert be.check_device_error() == 0


@pytest.mark.parametrize("reqs,max_new,d", WIDE + [([(1500, 1)] * 30, 1, 64), ([(1500, 2)] * 30, 2, 128)])
@pytest.mark.parametrize("score", [0.0, 2.0, 5.0])
def test_the_largest_value_of_the_type_does_not_overflow(be, reqs, max_new, d, score):
    """A weight of less than 1 times 3.4e38, its score above those before it: finite, as the sum divided is."""
    case = paged_case(127, 4, 2, d, 16, reqs, 0, stale=0.0)
    case[0][..., 5] = 1.0
    for i, (cached, _) in enumerate(reqs):
        p, o = at_key(case, i, min(200, cached) - 3)
        case[1][p, :, o, 5] = np.float32(score * d ** 0.5)
        case[2][p, :, o, 5] = np.float32(3.4e38)
    check_bound(be, case, d ** -0.5, max_new)


def sizes(rng, shape, kind, decades):
    """Factors up to 10^decades either way: none; some positions; some channels; some numbers; zero positions; zero numbers; one for all."""
    n, d = shape[0], shape[-1]
    some = lambda size, part: np.where(rng.random(size) < part, rng.uniform(-decades, decades, size), 0.0)  # noqa: E731
    f = {0: np.zeros(1), 1: some(n, rng.choice([0.02, 0.2, 0.6])).reshape(-1, *[1] * (len(shape) - 1)), 2: some(d, rng.choice([0.03, 0.3, 0.7])),
         3: some(shape, rng.choice([0.001, 0.01, 0.3])), 6: rng.uniform(-decades, decades, 1)}
    if kind == 4: return (rng.random(n) < 0.8).astype(np.float64).reshape(-1, *[1] * (len(shape) - 1))
    if kind == 5: return (rng.random(shape) < 0.5).astype(np.float64)
    return 10.0 ** f[kind]


@pytest.mark.parametrize("seed", range(24))
def test_numbers_far_apart_at_random(be, seed):
    """Groups of four adjacent head dims count as their largest number, which is what the tensor-core kernel promises."""
    rng = np.random.default_rng(1000 + seed)
    done = 0
    while done < 4:
        d, kvh, g, page = int(rng.choice([4, 8, 16, 20, 48, 64, 64])), int(rng.choice([1, 2])), int(rng.choice([1, 2, 4, 8])), int(rng.choice([1, 4, 5, 16]))
        reqs = [(int(rng.integers(0, 300)), int(rng.choice([1, 3, 20, 70]))) for _ in range(int(rng.integers(1, 3)))]
        q, kc, vc, table, q_start, kv_len = paged_case(int(rng.integers(1 << 30)), g * kvh, kvh, d, page, reqs, 1, stale=float(rng.choice([0.0, np.nan, 3e38])))
        decades, scale = float(rng.choice([3, 6, 12, 25])), float(rng.choice([d ** -0.5, 1.0, 0.01]))
        kinds = rng.integers(0, 7, 3)
        q = (q * sizes(rng, q.shape, int(kinds[0]), decades)).astype(np.float32)
        largest = 0.0
        for x, kind in ((kc, int(kinds[1])), (vc, int(kinds[2]))):
            for i, n in enumerate(kv_len):
                at = np.arange(n)
                part = x[table[i, at // page], :, at % page]
                part = np.clip(part * sizes(rng, part.shape, kind, decades), -3e38, 3e38).astype(np.float32)
                x[table[i, at // page], :, at % page] = part
                if x is kc: largest = max(largest, float(np.abs(part).max()))
        case = [q, kc, vc, table, q_start, kv_len]
        with np.errstate(over="ignore"):
            if float(np.abs(q).max()) * largest * d * max(1.5 * scale, 1.0) > 1e37 or np.abs(attend_bound(*case, scale)[0]).max() > 1e36:
                continue  # scores or sums that F32 does not hold
        done += 1
        check_bound(be, case, scale, max(x for _, x in reqs), fours)


@pytest.mark.parametrize("reqs,max_new,d", WIDE)
@pytest.mark.parametrize("what", ["k 1e8, q 1e-8", "q 1e8, k 1e-8", "q 1e12, k 0", "v 1e8", "v 1e20", "v zeros of the weightiest key", "v column of zeros",
                                  "v 1e36", "v 1e-36", "k zeros", "rows of q far apart", "four of k 1e-7", "four of v 1e-7", "four of q 1e-7",
                                  "four of all 1e-7", "half of v 1e-20", "half of q and k 1e-9", "zeros at the end", "v tiny and large"])
def test_channels_of_sizes_far_apart(be, reqs, max_new, d, what):
    q, kc, vc, *rest = paged_case(107, 4, 2, d, 16, reqs, 0, stale=0.0)
    case = [q, kc, vc, *rest]
    if what.startswith("k 1e8"): kc[..., 5] *= np.float32(1e8); q[..., 5] *= np.float32(1e-8)
    if what.startswith("q 1e8"): q[..., 5] *= np.float32(1e8); kc[..., 5] *= np.float32(1e-8)
    if what.startswith("q 1e12"): q[..., 5] *= np.float32(1e12); kc[..., 5] = 0
    if what == "v 1e8": vc[..., 5] *= np.float32(1e8)
    if what == "v 1e20": vc[..., 5] *= np.float32(1e20)
    if what == "v column of zeros": vc[..., 4:8] = 0
    if what == "v 1e36": vc *= np.float32(1e36)
    if what == "v 1e-36": vc *= np.float32(1e-36)
    if what == "k zeros": kc[rest[0][0, 0], :, 3:9] = 0; kc[..., 8:12] = 0
    if what.startswith("four of"):
        for x, name in ((q, "q"), (kc, "k"), (vc, "v")):
            if name in what[8:] or "all" in what: x[..., 4:8] *= np.float32(1e-7)
    if what == "half of v 1e-20": vc[..., ::2] *= np.float32(1e-20)
    if what == "half of q and k 1e-9": q[..., d // 2:] *= np.float32(1e-9); kc[..., : d // 2] *= np.float32(1e-9)
    if what == "zeros at the end": q[..., -d // 4:] = 0; kc[..., -d // 4:] = 0; vc[..., -d // 4:] = 0
    if what == "v tiny and large": vc *= np.float32(10.0) ** np.linspace(-34, 30, d).astype(np.float32)
    if what == "rows of q far apart": q *= np.float32(2.0) ** -np.arange(len(q), dtype=np.float32)[:, None, None].clip(0, 60)
    if what.startswith("v zeros"):
        q[..., 5] = 1.0
        p, o = at_key(case, 0, 2)
        kc[p, :, o, 5], vc[p, :, o] = np.float32(40 * d ** 0.5), 0
    check_bound(be, case, d ** -0.5, max_new)


@pytest.mark.parametrize("reqs", [[(40, 1), (3, 1)], [(70, 100), (20, 3)]])
@pytest.mark.parametrize("shift", [0, 1])
def test_attention_of_strided_views(be, reqs, shift):
    """q out of a fused product; caches stored position-major with other data between; shift leaves 16-byte alignment."""
    h, kvh, d, page = 4, 2, 16, 4
    q, kc, vc, table, q_start, kv_len = paged_case(37, h, kvh, d, page, reqs, 0, stale=0.0)
    rows, pages = len(q), len(kc)
    fused = rnd(1, rows, (h + 2 * kvh) * d + shift)
    fused[:, shift:shift + h * d] = q.reshape(rows, -1)
    tq = be.from_host(fused)
    tq.rank, tq.offset = 3, shift
    for i, (n_, s_) in enumerate(((rows, fused.shape[1]), (h, d), (d, 1))):
        tq.dims[i], tq.strides[i] = n_, s_
    raw = rnd(2, 2, pages, page, kvh + 1, d + shift)
    raw[0, :, :, :kvh, shift:], raw[1, :, :, :kvh, shift:] = kc.transpose(0, 2, 1, 3), vc.transpose(0, 2, 1, 3)
    store = be.from_host(raw)
    caches = []
    for i in range(2):
        r = store.copy_desc()
        r.rank, r.offset = 4, i * store.strides[0] + shift
        for a, (n_, s_) in enumerate(((pages, store.strides[1]), (kvh, store.strides[3]), (page, store.strides[2]), (d, 1))):
            r.dims[a], r.strides[a] = n_, s_
        caches.append(r)
    tt = strided(be.from_host(np.repeat(table, 2, 1)), 1, 2)
    ts = strided(be.from_host(np.repeat(q_start, 2)), 0, 2)
    tl = strided(be.from_host(np.repeat(kv_len, 2)), 0, 2)
    ref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.25)
    got = attend(be, tq, *caches, tt, ts, tl, 0.25)
    check_attention(ref, got, d, 200, np.abs(vc).max(), most, rms)
    assert be.check_device_error() == 0


def test_attention_over_shared_pages(be):
    """Two requests whose tables name the same prefix pages (a shared prompt)."""
    q, kc, vc, table, q_start, kv_len = paged_case(41, 4, 2, 64, 16, [(64, 2), (64, 1)])
    table[1, :4] = table[0, :4]
    ref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.125)
    check_attention(ref, attend(be, q, kc, vc, table, q_start, kv_len, 0.125), 64, 70, np.nanmax(np.abs(vc)), most, rms)


@pytest.mark.parametrize("reqs", [[(40, 1), (3, 1)], [(70, 100), (20, 3)]])
@pytest.mark.parametrize("page_id", [-1.0, 1e6, 0.5, float("nan"), float("inf")])
def test_wrong_page_ids_are_not_attended(be, reqs, page_id):
    q, kc, vc, table, q_start, kv_len = paged_case(43, 4, 2, 64, 16, reqs, 0, stale=0.0)
    wrong = table.astype(np.float32)
    wrong[0, 1] = page_id  # positions 16..31 of request 0
    got = attend(be, q, kc, vc, wrong, q_start, kv_len, 0.125)
    with pytest.raises(DeviceTimeoutError):
        be.check_device_error()
    # the definition without those keys: a score of -1e30 in their place
    far = kc.copy()
    ref = np.zeros(q.shape)
    for r in range(len(q)):
        i = int(np.searchsorted(q_start, r, "right")) - 1
        p = int(kv_len[i] - (q_start[i + 1] - q_start[i]) + r - q_start[i])
        at = [j for j in range(p + 1) if not (i == 0 and 16 <= j < 32)]
        for h in range(4):
            k = np.array([far[table[i, j // 16], h // 2, j % 16] for j in at], np.float64)
            v = np.array([vc[table[i, j // 16], h // 2, j % 16] for j in at], np.float64)
            w = np.exp(k @ q[r, h].astype(np.float64) * 0.125)
            ref[r, h] = w @ v / w.sum()
    most = np.abs(q).max() * np.abs(kc).max() * 64 * 0.125
    check_attention(ref, got, 64, 170, np.abs(vc).max(), most, most)


@pytest.mark.parametrize("start,length,max_new", [([0, 3, 2], [8, 8], 0), ([0, 1, 9], [8, 8], 0), ([-1, 1, 2], [8, 8], 0), ([0, 1, 2], [8, 1000], 0),
                                                  ([0, 1, 2], [8, -1], 0), ([0, 1.5, 2], [8, 8], 0), ([0, 1, 3], [8, 8], 1),
                                                  ([0, 1, 2], [float("nan"), 8], 0)])
def test_contradicting_requests_set_the_error_flag(be, start, length, max_new):
    """Wrong row or length values: the error flag; a request whose values are right is computed."""
    q, kc, vc, table, _, _ = paged_case(47, 4, 2, 64, 16, [(7, 1), (7, 1)], 2, stale=0.0)
    got = attend(be, q, kc, vc, table, np.array(start, np.float32), np.array(length, np.float32), 0.125, max_new)
    with pytest.raises(DeviceTimeoutError):
        be.check_device_error()
    if start[:2] == [0, 1] and length[0] == 8:
        ref, most, rms = attend_ref(q[:1], kc, vc, table[:1], [0, 1], [8], 0.125)
        check_attention(ref, got[:1], 64, 8, np.abs(vc).max(), most, rms)


def test_attention_refusals(be):
    d = 16
    base = dict(q=rnd(1, 3, 4, d), kc=rnd(2, 5, 2, 4, d), vc=rnd(3, 5, 2, 4, d), table=[[0, 1], [2, 3]], start=[0, 1, 3], length=[4, 5])

    def call(max_new=0, **kw):
        t = [x if isinstance(x, cabi.PaiTensor) else be.from_host(np.asarray(x, np.float32)) for x in (base | kw).values()]
        return be.sdpa_paged(*t, 0.25, max_new)

    call()
    for kw in (dict(start=[0, 3]), dict(length=[4]), dict(q=rnd(1, 3, 3, d)), dict(q=rnd(1, 3, 4, 8)), dict(vc=rnd(3, 5, 2, 4, 8)), dict(q=rnd(1, 3, d)),
               dict(table=[0, 1]), dict(kc=rnd(2, 5, 4, d)), dict(kc=rnd(2, 0, 2, 4, d)), dict(vc=cabi.transpose(be.from_host(rnd(3, 2, 5, 4, d)), 0, 1))):
        with pytest.raises(ArgumentError):
            call(**kw)
    with pytest.raises(OutOfRangeError):
        call(max_new=-1)
    wide = dict(q=rnd(1, 3, 4, 130), kc=rnd(2, 5, 2, 4, 130), vc=rnd(3, 5, 2, 4, 130))
    with pytest.raises(UnsupportedError):
        call(**wide)
    turned_ = [cabi.transpose(be.from_host(rnd(s, 5, 2, d, 4)), 2, 3) for s in (1, 2)]
    with pytest.raises(UnsupportedError):
        call(kc=turned_[0], vc=turned_[1])
    with pytest.raises(UnsupportedError):
        call(q=cabi.transpose(be.from_host(rnd(1, 3, d, 4)), 1, 2))
    with pytest.raises(UnsupportedError):  # 2^24 positions and more per request
        call(table=cabi.broadcast_to(be.from_host(np.zeros((1, 1), np.float32)), (2, (1 << 22) + 1)))


@pytest.mark.parametrize("new", [3, 40])
def test_a_contradicting_row_range_leaves_the_other_requests_rows(be, new):
    """q_start falls behind the first request's end: its last rows are its own, not rows behind the last request."""
    q, kc, vc, table, _, _ = paged_case(83, 4, 2, 64, 16, [(70, new), (7, 1)], 2, stale=0.0)
    start = np.array([0, new, new - 2], np.float32)
    ref, most, rms = attend_ref(q[:new], kc, vc, table[:1], [0, new], [70 + new], 0.125)
    for _ in range(5):
        got = attend(be, q, kc, vc, table, start, [70.0 + new, 8.0], 0.125, new)
        check_attention(ref, got[:new], 64, 70 + new, np.abs(vc).max(), most, rms)
        with pytest.raises(DeviceTimeoutError):
            be.check_device_error()


def test_attention_refuses_more_query_rows_than_32_bits_count(be):
    """rows x H counts query rows in 32 bits: 2^24 rows of 128 heads would wrap to a negative row. A batch whose tables
    could hold 2^63 pieces of work and more is no error: its launch is bounded."""
    one = be.from_host(np.zeros((1, 1, 1), np.float32))
    kc, vc = be.from_host(rnd(1, 2, 1, 4, 1)), be.from_host(rnd(2, 2, 1, 4, 1))
    with pytest.raises(UnsupportedError):
        be.sdpa_paged(cabi.broadcast_to(one, (1 << 24, 128, 1)), kc, vc, *map(be.from_host, ([[0.0]], [0.0, 0.0], [0.0])), 1.0, 1)
    with pytest.raises(UnsupportedError):
        be.sdpa_paged(cabi.broadcast_to(one, (1 << 24, 128, 1)), kc, vc, *map(be.from_host, ([[0.0]], [0.0, 0.0], [0.0])), 1.0, 0)
    kc, vc = be.from_host(rnd(1, 2, 64, 4, 1)), be.from_host(rnd(2, 2, 64, 4, 1))
    n, rows = 1 << 23, 1 << 20
    zero = be.from_host(np.zeros(1, np.float32))
    table = cabi.broadcast_to(be.from_host(np.zeros((1, 1), np.float32)), (n, 1 << 22))
    out = be.sdpa_paged(cabi.broadcast_to(one, (rows, 64, 1)), kc, vc, table, cabi.broadcast_to(zero, (n + 1,)), cabi.broadcast_to(zero, (n,)), 1.0, 0)
    assert not be.to_host(out).any()
    assert be.check_device_error() == 0


# ---------------------------------------------------------------- the operators together
class Server:
    """Steps of a server over one layer: plan, append, attend, with the dense float64 history beside it."""

    def __init__(self, be, h, kvh, d, page, pages, requests, max_pages, rows):
        self.be, self.h, self.kvh, self.d, self.page, self.rows = be, h, kvh, d, page, rows
        self.kc, self.vc = be.from_host(np.full((pages, kvh, page, d), np.nan, np.float32)), be.from_host(np.full((pages, kvh, page, d), np.nan, np.float32))
        self.table = be.from_host(np.full((requests, max_pages), -1, np.float32))
        self.ring = be.from_host(np.random.default_rng(0).permutation(pages).astype(np.float32))
        self.state, self.lengths = be.from_host(np.array([0, pages], np.float32)), be.from_host(np.zeros(requests, np.float32))
        self.new = be.from_host(np.zeros(requests, np.float32))
        self.qkv = be.from_host(np.zeros((rows, (h + 2 * kvh) * d), np.float32))
        self.cos, self.sin = tables(max_pages * page, d)
        self.tcos, self.tsin = be.from_host(self.cos), be.from_host(self.sin)
        self.history = [[] for _ in range(requests)]

    def ops(self):
        be, q, views = self.be, cabi.reshape(self.qkv, (self.rows, self.h + 2 * self.kvh, self.d)), []
        for at, n in ((0, self.h), (self.h, self.kvh), (self.h + self.kvh, self.kvh)):
            views.append(cabi.slice_view(q, 1, at, n))
        start, self.kv_len, slots, pos, self.next_state = be.paged_plan(self.lengths, self.new, self.table, self.ring, self.state, self.page, self.rows)
        rq = be.paged_rope_append(*views, self.tcos, self.tsin, pos, slots, self.kc, self.vc)
        return be.sdpa_paged(rq, self.kc, self.vc, self.table, start, self.kv_len, 1 / np.sqrt(self.d), 0)

    def expected(self, new, qkv):
        out, at, most = np.zeros((self.rows, self.h, self.d)), 0, 0.0
        x = qkv.reshape(self.rows, -1, self.d)
        for i, n in enumerate(new):
            if n < 0:
                self.history[i] = []
            for t in range(at, at + max(0, n)):
                p = [len(self.history[i])]
                turn = lambda y: turned(y[None], self.cos[p], self.sin[p])[0].astype(np.float64)  # noqa: E731
                self.history[i].append((turn(x[t, self.h:self.h + self.kvh]), x[t, self.h + self.kvh:].astype(np.float64)))
                q = turn(x[t, :self.h])
                for j in range(self.h):
                    k = np.array([kv[0][j // (self.h // self.kvh)] for kv in self.history[i]])
                    v = np.array([kv[1][j // (self.h // self.kvh)] for kv in self.history[i]])
                    w = np.exp(k @ q[j] / np.sqrt(self.d))
                    most = max(most, float((np.abs(k) @ np.abs(q[j])).max() / np.sqrt(self.d)))
                    out[t, j] = w @ v / w.sum()
            at += max(0, n)
        return out, most


STEPS = [[20, 3, 0], [1, 30, 7], [1, 1, 1], [-1, 1, 1], [0, 5, 1], [9, -1, 1], [1, 40, -1], [1, 1, 2], [70, 1, 1], [1, 1, 1]]


def run_steps(server, be, step):
    rng = np.random.default_rng(5)
    for n, new in enumerate(STEPS):
        qkv = rng.standard_normal((server.rows, (server.h + 2 * server.kvh) * server.d)).astype(np.float32)
        be.copy(be.from_host(np.array(new, np.float32)), server.new)
        be.copy(be.from_host(qkv), server.qkv)
        got = step(n)
        ref, most = server.expected(new, qkv)
        check_attention(ref, got, server.d, 130, np.abs(qkv).max(), most, most)
        assert be.to_host(server.lengths).tolist() == [float(len(h)) for h in server.history]


def test_a_server_runs_steps_of_joining_and_ending_requests(be):
    """Chunks, single tokens, requests that end and whose pages later ones take: every step against the dense history."""
    s = Server(be, 4, 2, 16, 8, 20, 3, 16, 84)

    def step(n):
        out = be.to_host(s.ops())
        s.lengths, s.state = s.kv_len, s.next_state
        return out

    run_steps(s, be, step)
    assert be.check_device_error() == 0
    held = sum(ceil_div(len(h), 8) for h in s.history)
    assert be.to_host(s.state)[1] == 20 - held


@pytest.mark.gpu
@pytest.mark.parametrize("h,kvh,d", [(4, 2, 16), (8, 2, 64)])
def test_a_captured_step_replays_for_every_later_one(cuda, h, kvh, d):
    """One step captured as a graph, its lengths and ring state carried over inside it; eager calls of another shape
    run between the replays."""
    s = Server(cuda, h, kvh, d, 8, 20, 3, 16, 84)
    other = paged_case(53, 8, 2, 64, 16, [(300, 257), (5, 1)])
    oref, omost, orms = attend_ref(*other, 0.125)
    graph, out = None, None

    def carried():
        r = s.ops()
        cuda.copy(s.kv_len, s.lengths)
        cuda.copy(s.next_state, s.state)
        return r

    def step(n):
        nonlocal graph, out
        if n == 0:
            return cuda.to_host(carried())
        if n == 1:
            cuda.graph_begin()
            out = carried()
            graph = cuda.graph_end()
        cuda.graph_launch(graph)
        got = cuda.to_host(out)
        check_attention(oref, attend(cuda, *other, 0.125), 64, 600, np.nanmax(np.abs(other[2])), omost, orms)
        return got

    run_steps(s, cuda, step)
    assert cuda.check_device_error() == 0
    cuda.graph_destroy(graph)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(cuda):
    """Caches of more than 2^31 elements, the requests in their last pages."""
    pages, kvh, page, d, h = 16600, 8, 256, 64, 16
    assert pages * kvh * page * d > 1 << 31
    kc, vc = cuda.allocate((pages, kvh, page, d)), cuda.allocate((pages, kvh, page, d))
    rng = np.random.default_rng(1)
    for new in (1, 130):
        rows, cached = new + 1, 300
        ids = [[pages - 1, pages - 3], [2, pages - 2]]
        length = [cached + new, 200]
        for i in range(2):  # fill through the append itself, at position 0: the rotation is the identity
            n = length[i]
            k, v, q = rnd(i, n, kvh, d), rnd(i + 5, n, kvh, d), rnd(i + 9, n, h, d)
            slots = np.array([ids[i][j // page] * page + j % page for j in range(n)])
            cuda.paged_rope_append(*map(cuda.from_host, (q, k, v, *tables(1, d), np.zeros(n), slots)), kc, vc)
            if i == 0:
                ks, vs = [k], [v]
            else:
                ks.append(k)
                vs.append(v)
        q = rng.standard_normal((rows, h, d)).astype(np.float32)
        # the same contents in small caches for the reference
        skc, svc = np.zeros((4, kvh, page, d), np.float32), np.zeros((4, kvh, page, d), np.float32)
        for i in range(2):
            for j in range(length[i]):
                skc[2 * i + j // page, :, j % page], svc[2 * i + j // page, :, j % page] = ks[i][j], vs[i][j]
        start = [0, new, new + 1]
        ref, most, rms = attend_ref(q, skc, svc, np.array([[0, 1], [2, 3]]), start, length, 0.125)
        got = attend(cuda, q, kc, vc, np.array(ids), np.array(start), np.array(length), 0.125, new)
        check_attention(ref, got, d, max(length), np.abs(svc).max(), most, rms)
    assert cuda.check_device_error() == 0


def test_host_runtime_binds_the_operators(request):
    """The same operators through _paihost.Backend, on the oracle library."""
    from conftest import ORACLE_LIB
    from projectai_b200 import _paihost as H

    request.getfixturevalue("oracle_lib")
    host_runtime(H.Backend(str(ORACLE_LIB), "oracle_", 0))


@pytest.mark.gpu
def test_host_runtime_binds_the_operators_on_cuda():
    import projectai_b200 as pai
    from projectai_b200 import _paihost as H

    host_runtime(H.Backend(str(pai.CUDA_LIB_PATH), "pai_", 0))


def host_runtime(be):
    q, kc, vc, table, q_start, kv_len = paged_case(59, 4, 2, 16, 4, [(9, 2), (0, 5)], 1, stale=0.0)
    lengths, new, ptable, ring, head, count = plan_inputs(6, [(9, 2), (0, 5)], 4)
    ref = PlanRef(lengths, new, ptable, ring, head, count, 4, 8)
    f = lambda a: be.from_host(np.array(a, np.float32))  # noqa: E731
    t = f(ptable)
    got = be.paged_plan(f(lengths), f(new), t, f(ring), f([head, count]), page_size=4, rows=8)
    for name, r in zip(("q_start", "kv_len", "slots", "positions", "state"), got):
        assert be.to_host(r).tolist() == list(map(float, getattr(ref, name)))
    assert np.array_equal(be.to_host(t), ref.table.astype(np.float32))
    k, v = rnd(1, 8, 2, 16), rnd(2, 8, 2, 16)
    cos, sin = tables(20, 16)
    slots, pos = np.array([0, 5, 9, -1, 2, 3, 4, 1]), np.arange(8)
    want = append_ref(q, k, v, cos, sin, pos, slots, kc, vc)
    tkc, tvc = f(kc), f(vc)
    rq = be.paged_rope_append(f(q), f(k), f(v), f(cos), f(sin), f(pos), f(slots), tkc, tvc)
    for a, b in zip(want, (rq, tkc, tvc)):
        assert np.array_equal(a, be.to_host(b))
    aref, most, rms = attend_ref(q, kc, vc, table, q_start, kv_len, 0.25)
    out = be.to_host(be.sdpa_paged(f(q), f(kc), f(vc), f(table), f(q_start), f(kv_len), 0.25))
    check_attention(aref, out, 16, 11, np.abs(vc).max(), most, rms)
    be.check_device_error()
