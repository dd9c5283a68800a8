"""Packed-batch operators (ops/packed.py) at the edges of their contracts: slices of a batch, arguments
that are refused, values on the device that no request should bring. Tolerances are those of
test_packed_gpu.py, whose cases and 64-bit statements are used here."""
import pytest
import torch

from test_packed_gpu import DEV, Case, _done, _i, _layout_plain, _layout_run, _packed

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------ slices of a batch
def _two_groups(prefixes, paged=True):
    """Two groups of requests, each with a pool and a prefix of its own, whose tokens share one batch."""
    a = Case([3, 1, 40], [9, 300, 40], 4, 2, 64, prefix=prefixes[0], seed=61, paged=paged)
    b = Case([1, 70, 5], [700, 90, 5], 4, 2, 64, prefix=prefixes[1], seed=62, paged=paged)
    n = a.N
    q = torch.cat([a.q, b.q])
    o = torch.full_like(q, 7.0)
    lse = torch.full((q.shape[0], 4), 7.0, device=DEV)
    start = _i(a.start + [n + s for s in b.start[1:]])
    for c, rows, at in ((a, slice(0, n), slice(0, 4)), (b, slice(n, None), slice(3, 7))):
        c.o, c.lse, c.at = o[rows], lse[rows], start[at]

    def run(c):
        P, kw = _packed(), dict(q_start=c.at, kv_len=_i(c.own), heads=4, kv_heads=2, head_dim=64, table=c.table, lse=lse)
        if c.prefix:
            P.shared_prefix_attention(q, c.k, c.v, o, prefix_table=c.prefix_table, prefix_len=c.prefix, **kw)
        else:
            P.packed_attention(q, c.k, c.v, o, k_start=c.k_start, **kw)
        _done()

    return a, b, run


@pytest.mark.parametrize("prefixes", [(200, 1000), (1000, 130), (0, 500), (500, 0), (0, 0)])
def test_groups_of_one_batch(prefixes):
    """Each call leaves the other group's rows alone, whichever comes first."""
    for order in (0, 1):
        a, b, run = _two_groups(prefixes)
        first, second = (b, a) if order else (a, b)
        run(first)
        assert bool((second.o == 7).all()) and bool((second.lse == 7).all())
        kept, kept_lse = first.o.clone(), first.lse.clone()
        run(second)
        assert torch.equal(first.o, kept) and torch.equal(first.lse, kept_lse)
        for c in (a, b):
            c.check()


def test_slice_without_requests():
    a, b, run = _two_groups((200, 300))
    b.at, b.own = b.at[:1], []
    run(b)
    assert bool((a.o == 7).all()) and bool((b.o == 7).all())


# ------------------------------------------------------------------------------------ after an error
@pytest.mark.parametrize("prefix", [0, 900])
def test_no_rows_are_joined_after_an_error(prefix):
    """An error that a kernel has recorded (its rows' parts may be missing): rows that would be joined stay
    as they are, the host learns of it, and the next call is right."""
    from appcorr_b200.ops.native import check_errors, err_word

    c = Case([1], [6001], 28, 4, 128, prefix=prefix, seed=67)  # one tile a key head, cut over all SMs
    err_word(torch.device(DEV)).fill_(2)
    P, kw = _packed(), dict(q_start=_i(c.start), kv_len=_i(c.own), heads=28, kv_heads=4, head_dim=128, table=c.table, lse=c.lse)
    if prefix:
        P.shared_prefix_attention(c.q, c.k, c.v, c.o, prefix_table=c.prefix_table, prefix_len=prefix, **kw)
    else:
        P.packed_attention(c.q, c.k, c.v, c.o, **kw)
    torch.cuda.synchronize()
    assert bool((c.o == 7).all()) and bool((c.lse == 7).all())
    with pytest.raises(RuntimeError, match="MMA wait timed out"):
        check_errors(torch.device(DEV))
    c.run()
    c.check()


# ------------------------------------------------------------------------------------ arguments
@pytest.mark.parametrize("prefix", [0, 200])
def test_attention_refuses_scales_that_order_no_scores(prefix):
    c = Case([2, 40], [2, 300], 4, 2, 64, prefix=prefix, seed=71)
    for scale in (0.0, -0.125, 1e-60, 1e60, float("nan"), float("inf")):  # 1e-60 and 1e60 are 0 and infinite in fp32
        with pytest.raises(RuntimeError, match="scale must be positive and finite"):
            c.run(scale=scale)
    assert bool((c.o == 7).all())
    c.run(scale=1e-30)  # every visible key alike
    c.check(scale=1e-30)


def _layout_args(B=3, N=5, W=4):
    e = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731
    return dict(q_len=e(B), past=e(B), table=e(B, W), free_pages=e(9), free_start=e(1), q_start=e(B + 1), kv_len=e(B), rows=e(N), req=e(N),
                pos=e(N), free_next=e(2))


LAYOUT_IN, LAYOUT_OUT = ("q_len", "past", "free_pages", "free_start", "table"), ("q_start", "kv_len", "rows", "req", "pos", "free_next")


def _layout_call(a):
    _packed().packed_layout(*(a[k] for k in ("q_len", "past", "table", "free_pages", "free_start")), **{k: a[k] for k in LAYOUT_OUT})


def _in_one_buffer(a, first, second, gap):
    """The two arguments as views of one buffer, the second `gap` values after the first one's begin."""
    n, m = a[first].numel(), a[second].numel()
    buf = torch.zeros(n + m + gap + 8, dtype=torch.int32, device=DEV)
    return {**a, first: buf[:n].view(a[first].shape), second: buf[gap:gap + m].view(a[second].shape)}


@pytest.mark.parametrize("out", LAYOUT_OUT)
def test_layout_refuses_outputs_in_place_of_other_arguments(out):
    for other in LAYOUT_IN + LAYOUT_OUT:
        if other == out:
            continue
        a = _layout_args()
        for first, second in ((out, other), (other, out)):
            for gap in (0, a[first].numel() - 1):  # the same place; one value in common
                with pytest.raises(RuntimeError, match="must not lie in the place of"):
                    _layout_call(_in_one_buffer(a, first, second, gap))
            _layout_call(_in_one_buffer(a, first, second, a[first].numel()))  # side by side
    _done()


def test_layout_overlaps_of_the_table():
    """What lies between the table's rows or behind those that are used is no part of it."""
    buf = torch.zeros(6, 9, dtype=torch.int32, device=DEV)
    a = _layout_args() | dict(table=buf[:, :4])
    _layout_call(a | dict(kv_len=buf[1, 4:7], q_start=buf[2, 5:9], free_next=buf[3, :2], q_len=buf[4, :3], past=buf[0, 6:9]))
    for kw in (dict(kv_len=buf[1, 3:6]), dict(q_start=buf[1, 6:10].new_zeros(0).set_(buf.untyped_storage(), 15, (4,))), dict(past=buf[2, :3]),
               dict(free_pages=buf.view(-1)[40 - 22:40 - 22 + 9]), dict(free_next=buf[0, 3:5]),
               dict(table=torch.zeros(4, dtype=torch.int32, device=DEV).expand(3, 4))):
        with pytest.raises(RuntimeError, match="must not lie in the place of|overlap"):
            _layout_call(a | kw)
    one = _layout_args(B=1) | dict(table=buf[:1, :9])
    _layout_call(one | dict(kv_len=buf[1, :1]))
    _done()


# ------------------------------------------------------------------------------------ values on the device
def test_layout_pages_without_rows():
    """A page number whose rows pass 32 bits is no page: its tokens get row -1, not some other page's row."""
    q, past = [4, 2, 1, 260, 3], [127, 200, 0, 0, 253]
    table = [[1 << 24, 5, 5], [3, 1 << 25, 5], [5, 5, 5], [5, 5, 5], [5, (1 << 24) - 1, 5]]
    free = [(1 << 30) + 1, 1 << 24, 7, -9]
    got = _layout_run(q, past, table, free, 0)
    want = _layout_plain(q, past, table, free, 0)
    want["rows"] = [r if r < 1 << 31 else -1 for r in want["rows"]]
    assert want["rows"].count(-1) == 4 + 2 + 1 + 132 and want["rows"][-1] == (1 << 31) - 1
    assert got == want


TOP = (1 << 31) - 1


@pytest.mark.parametrize("past", [TOP, TOP - 1, TOP - 126, TOP - 127, TOP - 128, TOP - 199, TOP - 200, TOP - 201, 1 << 30])
def test_layout_lengths_whose_sum_passes_32_bits(past):
    """Such requests get neither pages nor rows; those beside them are laid out, and nothing else is written."""
    q, pasts = [3, 200, 130], [126, past, 5]
    buf = torch.full((3, 3, 4), -7, dtype=torch.int32, device=DEV)
    buf[1, :, 0] = _i([20, 21, 22])
    out = {k: torch.full((n,), 77, dtype=torch.int32, device=DEV) for k, n in (("q_start", 4), ("kv_len", 3), ("rows", 333), ("req", 333), ("pos", 333), ("free_next", 2))}
    _packed().packed_layout(_i(q), _i(pasts), buf[1], _i([5, 6, 7]), _i([0]), **out)
    _done()
    want_kv = [129, min(past + 200, TOP), 135]
    blocks = -(-(past + 200) // 128) - -(-past // 128)
    assert out["q_start"].tolist() == [0, 3, 203, 333] and out["kv_len"].tolist() == want_kv
    assert buf[1].tolist() == [[20, 5, -7, -7], [21, -7, -7, -7], [22, 6, -7, -7]] and bool((buf[::2] == -7).all())
    assert out["rows"].tolist() == [20 * 128 + 126, 20 * 128 + 127, 5 * 128] + [-1] * 200 + list(range(22 * 128 + 5, 23 * 128)) + list(range(6 * 128, 6 * 128 + 7))
    assert out["req"].tolist() == [0] * 3 + [1] * 200 + [2] * 130
    assert out["pos"].tolist() == [126, 127, 128] + [min(past + i, TOP) for i in range(200)] + list(range(5, 135))
    assert out["free_next"].tolist() == [2, blocks]


def test_layout_lengths_of_the_largest_kind():
    """Lengths of 2^31 - 1 beside short ones, negative lengths: what fits the table and the batch is right."""
    out = {k: torch.full((n,), 77, dtype=torch.int32, device=DEV) for k, n in (("q_start", 4), ("kv_len", 3), ("rows", 40), ("req", 40), ("pos", 40), ("free_next", 2))}
    table = torch.full((3, 2), -7, dtype=torch.int32, device=DEV)
    _packed().packed_layout(_i([30, -5, TOP - 30]), _i([-1, 200, TOP]), table, _i([4, 5, 6]), _i([0]), **out)
    _done()
    assert out["q_start"].tolist() == [0, 30, 30, TOP] and out["kv_len"].tolist() == [30, 200, TOP]
    assert table.tolist() == [[4, -7], [-7, -7], [-7, -7]]
    assert out["rows"].tolist() == list(range(4 * 128, 4 * 128 + 30)) + [-1] * 10 and out["pos"][30:].tolist() == [TOP] * 10
    assert out["req"].tolist() == [0] * 30 + [2] * 10


# ------------------------------------------------------------------------------------ strides
def test_single_values_of_any_stride():
    """One value, or one column, has no inner stride (torch calls it contiguous whatever it is)."""
    one = lambda v: torch.full((1, 3), v, dtype=torch.int32, device=DEV)[:, 0]  # noqa: E731
    assert one(1).stride() == (3,) and one(1).is_contiguous() and _i([[1, 2]]).T[:1].stride(1) == 2
    a = _layout_args(B=1, N=2, W=1) | dict(q_len=one(2), past=one(3), kv_len=one(0), free_start=one(0), free_pages=one(9), table=_i([[4, 2]]).T[:1])
    _layout_call(a)
    _done()
    assert a["kv_len"].tolist() == [5] and a["rows"].tolist() == [4 * 128 + 3, 4 * 128 + 4] and a["pos"].tolist() == [3, 4]
    c = Case([2], [100], 4, 2, 64, seed=73)
    c.run(kv_len=one(100), table=torch.cat([c.table[:, :1]] * 2, 1).T[:1])
    c.check()
    c = Case([2], [100], 4, 2, 64, seed=73, prefix=5)
    c.prefix_table = torch.stack([c.prefix_table] * 2, 1)[:, 0]
    c.run(kv_len=one(100))
    c.check()


def test_rope_refuses_outputs_whose_rows_overlap():
    N, H, K, D = 4, 2, 1, 64
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device=DEV, dtype=dtype)  # noqa: E731

    def call(**kw):
        a = dict(qkv=z(N, (H + 2 * K) * D), q=z(N, H * D), k=z(N, K * D), v=z(N, K * D)) | kw
        _packed().qk_norm_rope(a["qkv"], z(1, N, dtype=torch.int32), z(D // 2, dtype=torch.float32), z(D // 2, dtype=torch.int32), a["q"],
                               a["k"], a["v"], heads=H, kv_heads=K, head_dim=D)

    for name, width in (("q", H * D), ("k", K * D), ("v", K * D)):
        for row in (0, 8, width - 8):
            with pytest.raises(RuntimeError, match="rows must not overlap"):
                call(**{name: z(N * width).as_strided((N, width), (row, 1))})
    call(qkv=z(1, (H + 2 * K) * D).expand(N, -1))  # read only: every token alike
    pool = z(N, 2, K * D)
    call(k=pool[:, 0], v=pool[:, 1])  # caches side by side in one pool
    _done()


# ------------------------------------------------------------------------------------ key lengths near 2^31
@pytest.mark.parametrize("paged,own", [(True, TOP), (True, TOP - 127), (False, TOP - 40)])
def test_attention_key_lengths_near_the_largest(paged, own):
    """Far more keys than there are rows: the missing ones are rows of zeros, as everywhere, and count. (A
    sum of 2^31 terms in fp32, 2^24 of them per block at the most, is off by less than 2^-11.)"""
    c = Case([1, 2], [200, 2], 4, 2, 64, seed=79, paged=paged)
    if paged:
        c.table = c.table[:, :2].contiguous()
        rest = int(c.rows[0][199]) + 1  # the second page's other rows are keys here
        c.k[rest:rest + 56], c.v[rest:rest + 56] = 0, 0
    else:
        c.k_start, c.k, c.v = _i([3, 0]), c.k[c.rows[0]].contiguous(), c.v[c.rows[0]].contiguous()
        c.rows = [torch.arange(3, 200, device=DEV), torch.arange(2, device=DEV)]
    c.run(kv_len=_i([own, 2]))
    k, v = (x[c.rows[0]].double().view(-1, 2, 64) for x in (c.k, c.v))
    for h in range(4):
        x = k[:, h // 2] @ c.q[0, h * 64:(h + 1) * 64].double() / 8
        total = x.exp().sum() + (own - x.numel())
        o, size = x.exp() @ v[:, h // 2] / total, x.exp() @ v[:, h // 2].abs() / total
        assert bool(((c.o[0, h * 64:(h + 1) * 64].double() - o).abs() <= 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2.0 ** -11) * size).all())
        assert abs(float(c.lse[0, h].double() - total.log())) <= 2.0 ** -11 + 2.0 ** -20 * 22


# ------------------------------------------------------------------------------------ streams
@pytest.mark.parametrize("prefix", [0, 1500])
def test_calls_on_two_streams_keep_apart(prefix):
    """Many calls in flight on two streams at once, every one into an output of its own that held NaN: the
    same bits as a call by itself. Nothing is uploaded or read in between."""
    P, calls = _packed(), 12
    cases = [Case([1] * 9, [700 + 111 * i for i in range(9)], 28, 4, 128, prefix=prefix, seed=s) for s in (83, 89)]
    want, args, outs = [], [], []
    for c in cases:
        c.run()
        c.check()
        want.append((c.o.clone(), c.lse.clone()))
        args.append(dict(q_start=_i(c.start), kv_len=_i(c.own), heads=28, kv_heads=4, head_dim=128, table=c.table) |
                    (dict(prefix_table=c.prefix_table, prefix_len=prefix) if prefix else {}))
        outs.append([(torch.full_like(c.o, float("nan")), torch.full_like(c.lse, float("nan"))) for _ in range(calls)])
    fn = P.shared_prefix_attention if prefix else P.packed_attention
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for i in range(calls):
        for c, a, out, s in zip(cases, args, outs, streams):
            with torch.cuda.stream(s):
                fn(c.q, c.k, c.v, out[i][0], lse=out[i][1], **a)
    _done()
    for (o, lse), out in zip(want, outs):
        for got, got_lse in out:
            assert torch.equal(got, o) and torch.equal(got_lse, lse)


# ------------------------------------------------------------------------------------ idle requests
def _slots(B, active, prefix):
    q_len, own = [0] * B, [300] * B
    for b, n, keys in active:
        q_len[b], own[b] = n, keys
    c = Case([n for n in q_len if n], [k for n, k in zip(q_len, own) if n], 4, 2, 64, prefix=prefix, seed=97)
    at, start, table = [b for b, n in enumerate(q_len) if n], [0], torch.full((B, c.table.shape[1]), 1 << 30, dtype=torch.int32)
    for n in q_len:
        start.append(start[-1] + n)
    table[at] = c.table.cpu()
    return c, dict(q_start=_i(start), kv_len=_i(own), table=table.to(DEV))


@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("B,active", [(40, (0, 39)), (700, (0, 31, 32, 33, 64, 699)), (700, (650,)), (3000, (1, 2998)), (33, (32,)), (34, (1, 33))])
def test_attention_between_idle_requests(B, active, prefix):
    """Requests without new tokens (whose tables hold no page) before, between and behind the active ones."""
    c, kw = _slots(B, [(b, 1 + 70 * (i & 1), 600 + 100 * i) for i, b in enumerate(active)], prefix)
    c.run(**kw)
    c.check()


@pytest.mark.parametrize("prefix", [0, 300])
def test_idle_requests_cost_little(prefix):
    """A few requests ahead of thousands of idle ones take no multiple of what as many, spread out, take."""
    times = []
    for active in (range(64), range(0, 16384, 256)):
        c, kw = _slots(16384, [(b, 1, 600) for b in active], prefix)
        c.run(**kw)
        ev = [torch.cuda.Event(enable_timing=True) for _ in range(6)]
        for e in ev:  # the outputs of the first call stay in c.o
            e.record()
            if prefix:
                _packed().shared_prefix_attention(c.q, c.k, c.v, c.o, prefix_table=c.prefix_table, prefix_len=prefix, heads=4, kv_heads=2, head_dim=64, **kw)
            else:
                _packed().packed_attention(c.q, c.k, c.v, c.o, heads=4, kv_heads=2, head_dim=64, **kw)
        torch.cuda.synchronize()
        times.append(min(a.elapsed_time(b) for a, b in zip(ev, ev[1:])))
        c.run(**kw)
        c.check()
    assert times[0] < 4 * times[1], times
