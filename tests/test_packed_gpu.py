"""Packed-batch operators (ops/packed.py) against plain 64-bit statements of their formulas: layouts
of a step, per-head norms with multi-axis rotation, packed causal attention, shared-prefix attention.

Tolerances. Outputs are rounded once to bf16 (relative 2^-8, half a unit of 8 significant bits). A rotated value is a cos - b sin with
fp32 sines, so its error is 2^-8 of itself plus a few 2^-23 of |a| + |b|. An attention output adds the
rounding of the probabilities to bf16 (2^-8 of each p_j |v_j|, no more than 2^-8 sum_j p_j |v_j| in
all), fp32 exponentials (relative 1e-4 of a probability at the most, 2^-12 taken) and fp32 scores: a sum
of D products is off by about sqrt(D) 2^-24 of s = scale sum_i |q_i k_i|, 2^-20 s taken over the keys
whose probability is not zero. |error| <= 2^-8 |o| + (2^-8 + 2^-12 + 2^-20 s) sum_j p_j |v_j|. A
log-sum-exp is off by the relative error of its sum and by the scores': 2^-11 + 2^-20 s."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 128


def _packed():
    from appcorr_b200.ops import packed

    return packed


def _done():
    from appcorr_b200.ops.native import check_errors

    torch.cuda.synchronize()
    check_errors(torch.device(DEV))


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------ layout
def _layout_plain(q, past, table, free, start):
    table = [list(r) for r in table]
    width, at, missing = len(table[0]), start, 0
    q_start, rows, req, pos = [0], [], [], []
    for b, (n, p) in enumerate(zip(q, past)):
        have, total = -(-p // PAGE), -(-(p + n) // PAGE)
        for blk in range(have, total):
            if blk >= width:
                missing += 1
                continue
            table[b][blk] = free[at] if at < len(free) else -1
            missing += at >= len(free)
            at += 1
        for i in range(p, p + n):
            page = table[b][i // PAGE] if i // PAGE < width else -1
            rows.append(page * PAGE + i % PAGE if page >= 0 else -1)
            req.append(b)
            pos.append(i)
        q_start.append(q_start[-1] + n)
    return dict(q_start=q_start, kv_len=[a + b for a, b in zip(q, past)], rows=rows, req=req, pos=pos, table=table,
                free_next=[min(at, max(len(free), start)), missing])


def _layout_run(q, past, table, free, start, pad=0):
    B, N = len(q), sum(q) + pad
    e = lambda n: torch.full((n,), 77, dtype=torch.int32, device=DEV)  # noqa: E731
    t = _i(table)
    out = dict(q_start=e(B + 1), kv_len=e(B), rows=e(N), req=e(N), pos=e(N), free_next=e(2))
    _packed().packed_layout(_i(q), _i(past), t, _i(free), _i([start]), **out)
    _done()
    return {k: v.tolist() for k, v in out.items()} | {"table": t.tolist()}


def _layout_case(B, longest, past_hi, seed):
    g = torch.Generator().manual_seed(seed)
    q = [int(v) for v in torch.randint(0, longest + 1, (B,), generator=g)]
    past = [int(v) for v in torch.randint(0, past_hi + 1, (B,), generator=g)]
    width = max(-(-(a + b) // PAGE) for a, b in zip(q, past)) + 1
    order = iter(torch.randperm(B * width + 50, generator=g).tolist())
    table = [[next(order) if blk < -(-p // PAGE) else -5 for blk in range(width)] for p in past]
    need = sum(-(-(a + b) // PAGE) - -(-b // PAGE) for a, b in zip(q, past))
    return q, past, table, [next(order) for _ in range(need + 4)]


@pytest.mark.parametrize("B,longest,past_hi", [(1, 1, 0), (1, 1, 127), (1, 0, 300), (3, 700, 300), (33, 5, 1000), (1024, 40, 500),
                                               (1025, 300, 129), (2500, 3, 128)])
@pytest.mark.parametrize("pad", [0, 37])
def test_layout(B, longest, past_hi, pad):
    q, past, table, free = _layout_case(B, longest, past_hi, B + longest)
    want = _layout_plain(q, past, table, free, 2)
    for k in ("rows", "req", "pos"):
        want[k] += [-1] * pad
    assert _layout_run(q, past, table, free, 2, pad) == want


@pytest.mark.parametrize("past,n", [(127, 1), (128, 1), (0, 128), (0, 129), (255, 2), (256, 0)])
def test_layout_page_edges(past, n):
    table = [[40, 41, 42, 43]]
    assert _layout_run([n], [past], table, [7, 8, 9], 1) == _layout_plain([n], [past], table, [7, 8, 9], 1)


def test_layout_short_of_pages_and_of_table():
    q, past = [200, 300, 0, 900], [100, 0, 5, 128]
    table = [[90 + 10 * b + i for i in range(5)] for b in range(4)]
    for free, start in (([1, 2, 3], 0), ([1, 2, 3], 2), ([1, 2, 3], 3), ([1], 5), (list(range(20)), 1)):
        want = _layout_plain(q, past, table, free, start)
        assert want["free_next"][1] > 0  # the last request needs more blocks than the table holds
        assert _layout_run(q, past, table, free, start) == want


def test_layout_steps_carry_on():
    """Steps chained through free_next give every page once."""
    P = _packed()
    B, W = 5, 6
    table = torch.full((B, W), -1, dtype=torch.int32, device=DEV)
    free = torch.randperm(64, device=DEV).to(torch.int32)
    past, start = torch.zeros(B, dtype=torch.int32, device=DEV), _i([0])
    e = lambda n: torch.empty(n, dtype=torch.int32, device=DEV)  # noqa: E731
    seen = []
    for step in range(4):
        q = _i([130, 1, 0, 64, 150][step:] + [130, 1, 0, 64, 150][:step])
        kv, nxt, rows = e(B), e(2), e(345)
        P.packed_layout(q, past, table, free, start, q_start=e(B + 1), kv_len=kv, rows=rows, req=e(345), pos=e(345), free_next=nxt)
        past, start = kv, nxt[:1]
        seen += rows.tolist()
    _done()
    assert nxt.tolist()[1] == 0
    assert len(set(seen)) == len(seen) == 4 * 345 and min(seen) >= 0
    held = [p for r, n in zip(table.tolist(), past.tolist()) for p in r[:-(-n // PAGE)]]
    assert held == list(dict.fromkeys(held)) and sorted(held) == sorted(free[:int(start)].tolist())


def test_layout_refusals():
    P = _packed()
    e = lambda *n: torch.zeros(*n, dtype=torch.int32, device=DEV)  # noqa: E731

    def call(**kw):
        a = dict(q_len=e(3), past=e(3), table=e(3, 4), free_pages=e(9), free_start=e(1), q_start=e(4), kv_len=e(3), rows=e(5), req=e(5),
                 pos=e(5), free_next=e(2)) | kw
        P.packed_layout(a.pop("q_len"), a.pop("past"), a.pop("table"), a.pop("free_pages"), a.pop("free_start"), **a)

    call()
    start = e(2)
    lens = e(3)
    for kw in (dict(past=lens, kv_len=lens), dict(q_len=lens, kv_len=lens), dict(past=e(2)), dict(table=e(2, 4)), dict(q_start=e(3)), dict(req=e(4)), dict(free_next=e(1)), dict(kv_len=e(3).long()),
               dict(rows=e(5).cpu()), dict(table=e(4, 3).t()), dict(free_start=start[:1], free_next=start)):
        with pytest.raises(RuntimeError):
            call(**kw)
    _done()


# ------------------------------------------------------------------------------------ norm + rotation
def _rope_plain(x, heads, dim, weight, eps, angle):
    x = x.double().view(x.shape[0], heads, dim)
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight.double()
    a, b = x[..., :dim // 2], x[..., dim // 2:]
    s, c = angle.sin()[:, None], angle.cos()[:, None]
    y = torch.cat([a * c - b * s, b * c + a * s], -1)
    size = torch.cat([a.abs() + b.abs()] * 2, -1)
    return y.flatten(1), size.flatten(1)


@pytest.mark.parametrize("N", [1, 5, 600, 2049, 8200])
@pytest.mark.parametrize("heads,kv_heads,dim", [(28, 4, 128), (3, 1, 64), (16, 16, 64), (1, 1, 128)])
@pytest.mark.parametrize("axes,norm", [(1, "none"), (3, "both"), (2, "q")])
def test_qk_norm_rope(N, heads, kv_heads, dim, axes, norm):
    if N > 600 and heads == 28:
        N = N // 2 + 1
    P = _packed()
    g = torch.Generator(device=DEV).manual_seed(N + heads)
    r = lambda *s: torch.randn(*s, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    wide = r(N, (heads + 2 * kv_heads) * dim + 16) * 3
    qkv = wide[:, 8:-8]  # a row stride of its own
    pos = torch.randint(0, 40000, (axes, N), generator=g, device=DEV, dtype=torch.int32)
    inv = (1e6 ** -(torch.arange(dim // 2, dtype=torch.float64) / (dim // 2))).float().to(DEV)
    axis = torch.randint(0, axes, (dim // 2,), generator=g, device=DEV, dtype=torch.int32)
    axis[3] = axes  # names no axis: not rotated
    qw = r(dim) if norm != "none" else None
    kw = r(dim) if norm == "both" else None
    pool = 2 * N + 3
    rows = torch.randperm(pool, generator=g, device=DEV)[:N].to(torch.int32)
    if N > 4:
        rows[::5] = -1
    kc, vc = r(pool, kv_heads * dim), r(pool, kv_heads * dim)
    k0, v0 = kc.clone(), vc.clone()
    q = torch.empty(N, heads * dim, device=DEV, dtype=torch.bfloat16)
    P.qk_norm_rope(qkv, pos, inv, axis, q, kc, vc, heads=heads, kv_heads=kv_heads, head_dim=dim, rows=rows, q_weight=qw, k_weight=kw, eps=1e-5)
    _done()
    full = torch.cat([pos, pos.new_zeros(1, N)]).double()
    angle = full[axis.long()].T * inv.double()
    H, K = heads * dim, kv_heads * dim
    wq, sq = _rope_plain(qkv[:, :H], heads, dim, qw, 1e-5, angle)
    wk, sk = _rope_plain(qkv[:, H:H + K], kv_heads, dim, kw, 1e-5, angle)
    tol = lambda w, s: 2.0 ** -8 * w.abs() + 16 * 2.0 ** -23 * s + 1e-30  # noqa: E731
    assert bool(((q.double() - wq).abs() <= tol(wq, sq)).all())
    keep = rows >= 0
    at = rows[keep].long()
    assert bool(((kc[at].double() - wk[keep]).abs() <= tol(wk, sk)[keep]).all())
    assert torch.equal(vc[at], qkv[:, H + K:][keep])
    k0[at], v0[at] = kc[at], vc[at]
    assert torch.equal(kc, k0) and torch.equal(vc, v0)  # no other cache row is written


def test_qk_norm_rope_in_place_and_without_rows():
    P = _packed()
    torch.manual_seed(0)
    N, H, K, D = 70, 4, 2, 64
    qkv = torch.randn(N, (H + 2 * K) * D, device=DEV).to(torch.bfloat16)
    pos = torch.arange(N, device=DEV, dtype=torch.int32)[None]
    inv = torch.rand(D // 2, device=DEV)
    axis = torch.zeros(D // 2, device=DEV, dtype=torch.int32)
    outs = []
    for place in (False, True):
        x = qkv.clone()
        q = x[:, :H * D] if place else torch.empty(N, H * D, device=DEV, dtype=torch.bfloat16)
        kc, vc = (torch.zeros(N, K * D, device=DEV, dtype=torch.bfloat16) for _ in range(2))
        P.qk_norm_rope(x, pos, inv, axis, q, kc, vc, heads=H, kv_heads=K, head_dim=D)
        outs.append((q.clone(), kc, vc))
    _done()
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    assert torch.equal(outs[0][2], qkv[:, (H + K) * D:])


def test_qk_norm_rope_row_offsets_past_32_bits():
    P = _packed()
    H, K, D = 1, 32, 128
    rows_n = (1 << 31) // (K * D) + 300  # the pool's last elements lie past 2^31
    kc = torch.zeros(rows_n, K * D, device=DEV, dtype=torch.bfloat16)
    vc = torch.zeros(rows_n, K * D, device=DEV, dtype=torch.bfloat16)
    x = torch.randn(3, (H + 2 * K) * D, device=DEV).to(torch.bfloat16)
    rows = _i([rows_n - 1, 5, rows_n])  # the last one lies outside: not written
    zero = torch.zeros(D // 2, device=DEV)
    P.qk_norm_rope(x, _i([[1, 2, 3]]), zero, zero.to(torch.int32), torch.empty(3, H * D, device=DEV, dtype=torch.bfloat16), kc, vc,
                   heads=H, kv_heads=K, head_dim=D, rows=rows)
    _done()
    for n, r in ((0, rows_n - 1), (1, 5)):
        assert torch.equal(kc[r], x[n, H * D:(H + K) * D]) and torch.equal(vc[r], x[n, (H + K) * D:])
    assert int(kc.any(1).sum()) == 2


def test_qk_norm_rope_refusals():
    P = _packed()
    N, H, K, D = 4, 2, 1, 64
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device=DEV, dtype=dtype)  # noqa: E731

    def call(head_dim=D, rows=None, q_weight=None, **kw):
        a = dict(qkv=z(N, (H + 2 * K) * D), pos=z(1, N, dtype=torch.int32), inv=z(D // 2, dtype=torch.float32),
                 axis=z(D // 2, dtype=torch.int32), q=z(N, H * D), k=z(N, K * D), v=z(N, K * D)) | kw
        P.qk_norm_rope(a["qkv"], a["pos"], a["inv"], a["axis"], a["q"], a["k"], a["v"], heads=H, kv_heads=K, head_dim=head_dim, rows=rows,
                       q_weight=q_weight)

    call()
    for kw in (dict(head_dim=96), dict(qkv=z(N, 5 * D)), dict(qkv=z(N, (H + 2 * K) * D, dtype=torch.float32)),
               dict(qkv=z(N, (H + 2 * K) * D + 1)[:, 1:]), dict(pos=z(1, N + 1, dtype=torch.int32)), dict(pos=z(1, N, dtype=torch.int64)),
               dict(inv=z(D, dtype=torch.float32)), dict(q=z(N - 1, H * D)), dict(k=z(N - 1, K * D)), dict(v=z(N, K * D).cpu()),
               dict(rows=z(N - 1, dtype=torch.int32)), dict(q_weight=z(D // 2))):
        with pytest.raises(RuntimeError):
            call(**kw)
    _done()


# ------------------------------------------------------------------------------------ attention
def _attend_plain(q, k, v, scale, seen):
    """q [t, D], k / v [n, D], seen [t, n] -> o, sum p |v|, log-sum-exp and the largest s (64 bits)."""
    x = (q.double() @ k.double().T) * scale
    x[~seen] = -math.inf
    m = x.amax(1, keepdim=True) if x.shape[1] else x.new_full((x.shape[0], 1), -math.inf)
    e = torch.where(seen, (x - m.clamp(min=-1e300)).exp(), torch.zeros_like(x))
    total = e.sum(1, keepdim=True)
    p = torch.where(total > 0, e / total.clamp(min=1e-300), torch.zeros_like(e))
    lse = torch.where(total > 0, m + total.log(), torch.full_like(m, -math.inf))
    s = torch.where(p > 1e-30, (q.double().abs() @ k.double().abs().T) * scale, torch.zeros_like(x)) if x.shape[1] else m
    return p @ v.double(), p @ v.double().abs(), lse[:, 0], s.amax(1).clamp(min=0)


class Case:
    """A packed batch with random pages; what lies past a request's keys in its last page, and every
    row that no request holds, is NaN."""

    def __init__(self, q_len, own, heads, kv_heads, dim, prefix=0, paged=True, seed=0, peak=1.0, pad=0, wide=False):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.q_len, self.own, self.heads, self.kv_heads, self.dim, self.prefix = q_len, own, heads, kv_heads, dim, prefix
        B, N = len(q_len), sum(q_len)
        r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
        start = [0]
        for n in q_len:
            start.append(start[-1] + n)
        self.start, self.N = start, N
        extra = 24 if wide else 0
        self.q = (r(N + pad, heads * dim + extra) * peak).to(torch.bfloat16)[:, :heads * dim]
        o = torch.full((N + pad, heads * dim + extra), 7.0, device=DEV, dtype=torch.bfloat16)
        self.o = o[:, :heads * dim]
        blocks = [-(-n // PAGE) for n in own]
        shared = -(-prefix // PAGE)
        if paged:
            pages = sum(blocks) + shared + 2
            place = torch.randperm(pages, generator=g, device=DEV)
            rows = pages * PAGE
            self.table = torch.full((B, max(blocks + [1]) + 1), 1 << 30, device=DEV, dtype=torch.int32)  # unused: no page at all
            self.rows = []
            at = 0
            for b, n in enumerate(blocks):
                mine = place[at:at + n]
                at += n
                self.table[b, :n] = mine.to(torch.int32)
                self.rows.append((mine[:, None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(-1)[:own[b]])
            mine = place[at:at + shared]
            self.prefix_table = mine.to(torch.int32)
            self.front = (mine[:, None] * PAGE + torch.arange(PAGE, device=DEV)).reshape(-1)[:prefix]
            self.k_start = None
        else:
            first = [5]
            for n in own:
                first.append(first[-1] + n + 3)
            rows = first[-1] + 1
            self.table, self.k_start = None, _i(first[:-1])
            self.rows = [torch.arange(first[b], first[b] + n, device=DEV) for b, n in enumerate(own)]
            self.front = torch.zeros(0, dtype=torch.long, device=DEV)
        held = torch.cat(self.rows + [self.front])
        self.k = torch.full((rows, kv_heads * dim + extra), math.nan, device=DEV, dtype=torch.bfloat16)[:, :kv_heads * dim]
        self.v = torch.full((rows, kv_heads * dim + extra), math.nan, device=DEV, dtype=torch.bfloat16)[:, :kv_heads * dim]
        self.k[held] = r(held.numel(), kv_heads * dim).to(torch.bfloat16)
        self.v[held] = r(held.numel(), kv_heads * dim).to(torch.bfloat16)
        self.lse = torch.full((N + pad, heads), 7.0, device=DEV)

    def run(self, **kw):
        P = _packed()
        a = dict(q_start=_i(self.start), kv_len=_i(self.own), heads=self.heads, kv_heads=self.kv_heads, head_dim=self.dim, table=self.table,
                 lse=self.lse) | kw
        if self.prefix:
            P.shared_prefix_attention(self.q, self.k, self.v, self.o, prefix_table=self.prefix_table, prefix_len=self.prefix, **a)
        else:
            P.packed_attention(self.q, self.k, self.v, self.o, k_start=self.k_start, **a)
        _done()
        return self.o

    def check(self, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        D, G = self.dim, self.heads // self.kv_heads
        for b, n in enumerate(self.q_len):
            lo, hi = self.start[b], self.start[b + 1]
            rows = torch.cat([self.front, self.rows[b]])
            last = self.prefix + self.own[b] - n + torch.arange(n, device=DEV)
            seen = (torch.arange(rows.numel(), device=DEV) <= last[:, None]) | (torch.arange(rows.numel(), device=DEV) < self.prefix)
            for h in range(self.heads):
                kv = slice(h // G * D, (h // G + 1) * D)
                w, size, lse, s = _attend_plain(self.q[lo:hi, h * D:(h + 1) * D], self.k[rows][:, kv], self.v[rows][:, kv], scale, seen)
                got = self.o[lo:hi, h * D:(h + 1) * D].double()
                bad = ~((got - w).abs() <= 2.0 ** -8 * w.abs() + (2.0 ** -8 + 2.0 ** -12 + 2.0 ** -20 * s[:, None]) * size + 1e-30)
                assert not bool(bad.any()), (b, h, bad.nonzero()[:3].tolist(), float((got - w).abs().max()))
                gl = self.lse[lo:hi, h].double()
                assert torch.equal(gl == -math.inf, lse == -math.inf), (b, h)
                fin = lse > -math.inf
                assert bool(((gl - lse).abs()[fin] <= 2.0 ** -11 + 2.0 ** -20 * s[fin]).all()), (b, h)
        assert bool((self.o[self.N:] == 7).all()) and bool((self.lse[self.N:] == 7).all())


HEADS = [(28, 4, 128), (4, 2, 64), (5, 5, 128), (16, 1, 64)]


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("q_len", [[1], [2], [127, 1, 129], [300, 0, 17, 1], [1, 1, 1, 1, 1, 1, 1], [700]])
def test_attention_prompts(heads, kv_heads, dim, paged, q_len):
    c = Case(q_len, list(q_len), heads, kv_heads, dim, paged=paged, seed=len(q_len))
    c.run()
    c.check()


@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("q_len,own", [([1], [1000]), ([1, 1, 1], [128, 129, 2047]), ([5, 1, 64], [900, 3, 200]), ([1], [6001]),
                                       ([33, 2], [33, 5000]), ([1] * 40, list(range(1, 2001, 50)))])
def test_attention_after_cached_tokens(heads, kv_heads, dim, q_len, own):
    c = Case(q_len, own, heads, kv_heads, dim, seed=7, wide=True, pad=3)
    c.run()
    c.check()


@pytest.mark.parametrize("heads,kv_heads,dim", [(28, 4, 128), (8, 8, 64), (3, 1, 128), (129, 1, 64), (160, 2, 128)])
def test_attention_head_groups(heads, kv_heads, dim):
    c = Case([3, 150], [260, 150], heads, kv_heads, dim, seed=3)
    c.run()
    c.check()


def test_attention_rows_without_keys():
    """More new tokens than keys (the first tokens see none), and requests with no keys at all."""
    c = Case([5, 3, 200, 1], [2, 0, 130, 0], 4, 2, 64, seed=5)
    c.run()
    c.check()
    assert bool((c.o[:3] == 0).all()) and bool((c.o[5:8] == 0).all())


@pytest.mark.parametrize("peak", [0.0, 30.0, 3000.0])
def test_attention_flat_and_peaked(peak):
    """Equal scores, and scores whose maximum moves by far more than an exponent holds."""
    for q_len, own in (([260], [260]), ([1, 1], [700, 3000])):
        c = Case(q_len, own, 4, 2, 128, seed=11, peak=peak)
        c.run()
        c.check()


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_attention_sorted_scores(order):
    """The running maximum grows with every key block, or never after the first."""
    c = Case([1, 200], [1500, 1500], 4, 2, 64, seed=13)
    ramp = torch.linspace(-40, 40, 1500, device=DEV)
    if order == "falling":
        ramp = ramp.flip(0)
    c.q[:] = 1.0
    for b in range(2):
        c.k[c.rows[b]] = (ramp[:, None] / 8).expand(-1, 128).to(torch.bfloat16)
    c.run()
    c.check()


def test_attention_scale_and_lowest_scores():
    """A scale of its own; scores near the lowest value of the type everywhere but on one key."""
    c = Case([1, 40], [300, 300], 4, 2, 64, seed=17)
    c.run(scale=0.5)
    c.check(scale=0.5)
    for b in range(2):
        c.k[c.rows[b]] = -1.5e36
        c.k[c.rows[b][:1]] = 0.25
    c.q[:] = 1.0
    c.run()
    c.check()


def test_attention_padded_tokens_and_strides():
    c = Case([4, 130], [20, 130], 28, 4, 128, seed=19, pad=60, wide=True)
    c.run()
    c.check()


def test_attention_on_another_stream_and_twice():
    """Calls on two streams at once keep their workspaces apart; a repeated call gives the same bits."""
    cases = [Case([1] * 9, [4000 + 111 * i for i in range(9)], 28, 4, 128, seed=s) for s in (23, 29)]
    first = [c.run().clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                _packed().packed_attention(c.q, c.k, c.v, c.o, q_start=_i(c.start), kv_len=_i(c.own), heads=28, kv_heads=4, head_dim=128,
                                           table=c.table, lse=c.lse)
    _done()
    for c, f in zip(cases, first):
        assert torch.equal(c.o, f)
        c.check()


def test_attention_many_requests():
    """More requests than one block has threads, most of them tiny, a few long."""
    g = torch.Generator().manual_seed(31)
    B = 1500
    q_len = [1 if int(v) else 0 for v in torch.randint(0, 9, (B,), generator=g)]
    own = [int(v) for v in torch.randint(1, 40, (B,), generator=g)]
    q_len[700], own[700], own[1499] = 300, 900, 2500
    c = Case(q_len, own, 2, 1, 64, seed=31)
    c.run()
    c.check()


# ------------------------------------------------------------------------------------ shared prefix
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("prefix", [1, 128, 1000])
@pytest.mark.parametrize("q_len,own", [([1], [1]), ([1, 1, 1], [40, 1, 300]), ([4] * 11, list(range(4, 400, 36))), ([70, 1, 300], [70, 0, 420])])
def test_shared_prefix(heads, kv_heads, dim, prefix, q_len, own):
    c = Case(q_len, own, heads, kv_heads, dim, prefix=prefix, seed=prefix)
    c.run()
    c.check()


@pytest.mark.parametrize("B,prefix", [(130, 700), (40, 5003), (2, 9000)])
def test_shared_prefix_long_and_wide(B, prefix):
    c = Case([1] * B, [1 + 7 * i for i in range(B)], 28, 4, 128, prefix=prefix, seed=B, pad=5, wide=True)
    c.run()
    c.check()


def test_shared_prefix_requests_without_own_keys():
    """kv_len 0: the prefix alone; rows ahead of their own keys still see the prefix."""
    c = Case([1, 3, 2], [0, 1, 0], 4, 2, 64, prefix=200, seed=41)
    c.run()
    c.check()


def test_shared_prefix_of_no_keys():
    c = Case([2, 1], [5, 300], 4, 2, 64, seed=43)
    P = _packed()
    P.shared_prefix_attention(c.q, c.k, c.v, c.o, q_start=_i(c.start), kv_len=_i(c.own), table=c.table,
                              prefix_table=torch.empty(0, dtype=torch.int32, device=DEV), prefix_len=0, heads=4, kv_heads=2, head_dim=64,
                              lse=c.lse)
    _done()
    c.check()


@pytest.mark.parametrize("heads,kv_heads,dim", [(2, 1, 64)])
def test_attention_pool_past_32_bits(heads, kv_heads, dim):
    """Cache elements past 2^31: pages at the end of a pool of 2^31 + elements."""
    pages = (1 << 31) // (PAGE * 4096) + 2
    k = torch.zeros(pages * PAGE, 4096, device=DEV, dtype=torch.bfloat16)
    v = torch.zeros(pages * PAGE, 4096, device=DEV, dtype=torch.bfloat16)
    c = Case([2], [200], heads, kv_heads, dim, seed=47)
    big = [pages - 1, pages - 2]
    rows = torch.cat([torch.arange(p * PAGE, (p + 1) * PAGE, device=DEV) for p in big])[:200]
    k[rows, :64], v[rows, :64] = c.k[c.rows[0]], c.v[c.rows[0]]
    c.k, c.v, c.rows, c.table = k[:, :64], v[:, :64], [rows], _i([big])
    c.run()
    c.check()


def test_attention_missing_pages_read_as_zeros():
    """Pages below zero or past the pool, and blocks past the table, are rows of zeros."""
    c = Case([1, 2], [300, 260], 4, 2, 64, seed=53)
    real = [r.clone() for r in c.rows]
    c.table[0, 1], c.table[1, 0] = -1, 1 << 29
    table = c.table[:, :2].contiguous()
    c.run(table=table)
    k, v = torch.zeros(1 + c.k.shape[0], 128, device=DEV, dtype=torch.bfloat16), torch.zeros(1 + c.k.shape[0], 128, device=DEV, dtype=torch.bfloat16)
    k[1:], v[1:] = c.k, c.v
    real = [r + 1 for r in real]
    real[0][128:], real[1][:128], real[1][256:] = 0, 0, 0
    c.k, c.v, c.rows = k, v, real
    c.check()


def test_attention_refusals():
    P = _packed()
    H, K, D = 4, 2, 64
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device=DEV, dtype=dtype)  # noqa: E731
    zi = lambda *s: z(*s, dtype=torch.int32)  # noqa: E731

    def call(prefix=False, **kw):
        a = dict(q=z(3, H * D), k=z(256, K * D), v=z(256, K * D), o=z(3, H * D), q_start=zi(3), kv_len=zi(2), heads=H, kv_heads=K,
                 head_dim=D, table=zi(2, 2)) | (dict(prefix_table=zi(2), prefix_len=200) if prefix else {}) | kw
        fn = P.shared_prefix_attention if prefix else P.packed_attention
        fn(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("o"), **a)

    call()
    call(prefix=True)
    for kw in (dict(head_dim=32), dict(heads=3), dict(q=z(3, H * D).float()), dict(q=z(3, H * D).cpu()), dict(q=z(3, 2 * H * D)[:, ::2]),
               dict(k=z(250, K * D)), dict(v=z(384, K * D)), dict(o=z(2, H * D)), dict(q_start=zi(2)), dict(kv_len=zi(2).long()),
               dict(table=zi(1, 2)), dict(table=None), dict(k_start=zi(2)), dict(table=zi(2, 2).t().contiguous().t()),
               dict(q=z(3, H * D + 4)[:, 4:]), dict(lse=z(3, H)), dict(lse=z(2, H, dtype=torch.float32)),
               dict(prefix=True, prefix_len=300), dict(prefix=True, prefix_len=-1), dict(prefix=True, prefix_table=zi(2).long())):
        with pytest.raises(RuntimeError):
            call(**kw)
    _done()
    empty = dict(q=z(0, H * D), o=z(0, H * D), q_start=zi(1), kv_len=zi(0), table=zi(0, 1))
    call(**empty)
    _done()
