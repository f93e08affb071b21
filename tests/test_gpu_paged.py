"""Operators on device data (androidllm_b200.paged) against their formulas in
64 bits.

Tolerances count roundings.  `half step` of a type is eps / 2 of the value
(fp16 2^-11, bf16 2^-8).
  append   computed in fp32 from at most four rounded products, then rounded
           once: half a step of the result plus 2^-20 of the head's largest
           value (cancelled products).
  attend   the output's half step; the weights' half step each, which moves a
           row by at most half a step of A = sum w |v| / sum w; scores are fp32
           sums of D products (error (D + 8) 2^-24 scale sum |q||k| =: d), a
           weight's relative error is 2 d + 2^-21 (exponential), and summing n
           terms in fp32 adds n 2^-24: all times A.  fp16 weights below 2^-14
           are off by up to 2^-25 absolutely: 2^-25 sum |v| / sum w.
  lse      d + n 2^-24 + 2^-21 of itself.
  verify   whole numbers, equal; p_draft from 32-bit exponentials: 1e-5.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from androidllm_b200 import ops, paged                  # noqa: E402
from androidllm_b200._lib import ALMError               # noqa: E402

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture()
def ctx():
    return ops.default_context(0, torch.cuda.current_stream().cuda_stream)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Batch:
    """A ragged batch over a scrambled page pool; what no sequence owns is NaN."""

    def __init__(self, rows, lens, page, kv_heads, dim, dtype, seed=0, tail=3, first=0, slots=None, extra_pages=4):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.gen, self.rows, self.lens, self.page, self.dim, self.hk, self.dt = g, rows, lens, page, dim, kv_heads, dtype
        start = [first]
        for r in rows:
            start.append(start[-1] + r)
        self.start, self.n_rows = start, start[-1] + tail
        need = [max(0, -(-n // page)) for n in lens]
        n_pages = sum(need) + extra_pages
        order = torch.randperm(n_pages, generator=g, device="cuda").tolist()
        width = max(need + [1]) + 1
        n_seq = len(rows)
        self.slot = list(range(n_seq)) if slots is None else slots
        table = torch.full((max(self.slot + [0]) + 1, width), -7, dtype=torch.int32)
        at = 0
        self.k = torch.full((n_pages, kv_heads, page, dim), float("nan"), device="cuda", dtype=dtype)
        self.v = self.k.clone()
        for s in range(n_seq):
            for i in range(need[s]):
                p = order[at]
                at += 1
                table[self.slot[s], i] = p
                live = min(page, lens[s] - i * page)
                self.k[p, :, :live] = (torch.randn(kv_heads, live, dim, generator=g, device="cuda") * 1.3).to(dtype)
                self.v[p, :, :live] = torch.randn(kv_heads, live, dim, generator=g, device="cuda").to(dtype)
        self.table = table.cuda()
        self.kv = paged.PagedKV(self.k, self.v)
        self.seqs = paged.SeqBatch(ints(start), ints(lens), self.table, n_rows=self.n_rows,
                                   max_rows=max(rows + [1]), slots=None if slots is None else ints(slots))

    def randn(self, *shape):
        return torch.randn(*shape, generator=self.gen, device="cuda").to(self.dt)

    def cached(self, s):
        """K, V (kv_heads, len, dim) of sequence s in 64 bits."""
        n = max(0, self.lens[s])
        pages = self.table[self.slot[s], :-(-n // self.page)].long()
        return tuple(x[pages].transpose(0, 1).reshape(self.hk, -1, self.dim)[:, :n].double() for x in (self.k, self.v))


def formula(b, q, scale, window=0, group=None):
    """out, lse and their tolerances (see above), in 64 bits; rows of no
    sequence are NaN."""
    heads = q.shape[1]
    group = heads // b.hk
    out = torch.full(q.shape, float("nan"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full(q.shape[:2], float("nan"), dtype=torch.float64, device="cuda")
    lse_tol = torch.zeros_like(lse)
    half = torch.finfo(q.dtype).eps / 2
    for s, n_new in enumerate(b.rows):
        lo, hi = b.start[s], b.start[s + 1]
        if n_new == 0:
            continue
        k, v = b.cached(s)
        n = k.shape[1]
        pos = b.lens[s] - n_new + torch.arange(n_new, device="cuda")
        j = torch.arange(n, device="cuda")
        seen = j[None] <= pos[:, None]
        if window:
            seen &= j[None] > pos[:, None] - window
        for h in range(heads):
            kh, vh = k[h // group], v[h // group]
            x = q[lo:hi, h].double()
            sc = (x @ kh.T) * scale
            d = (b.dim + 8) * 2.0 ** -24 * scale * (x.abs() @ kh.abs().T)
            d = torch.where(seen, d, 0.0).amax(1) if n else torch.zeros(n_new, device="cuda", dtype=torch.float64)
            sc = sc.masked_fill(~seen, -math.inf)
            none = ~seen.any(1)
            m = sc.amax(1) if n else torch.full((n_new,), -math.inf, device="cuda", dtype=torch.float64)
            m = torch.where(none, 0.0, m)
            w = torch.exp(sc - m[:, None])
            l = w.sum(1)
            ls = torch.where(none, 1.0, l)
            # a hidden position adds nothing, whatever its value is
            vz = torch.where(torch.isfinite(vh), vh, 0.0)
            o = (w @ vz) / ls[:, None]
            big = (w @ vz.abs()) / ls[:, None]
            out[lo:hi, h] = o
            rel = half + 2 * d + 2.0 ** -21 + (n + b.dim) * 2.0 ** -24
            tol[lo:hi, h] = half * o.abs() + rel[:, None] * big
            if q.dtype == torch.float16:
                tol[lo:hi, h] += 2.0 ** -25 * (seen.double() @ vz.abs()) / ls[:, None] + 2.0 ** -25
            lse[lo:hi, h] = torch.where(none, -math.inf, m + torch.log(ls))
            lse_tol[lo:hi, h] = d + n * 2.0 ** -24 + 2.0 ** -21 * (1 + torch.where(none, 0.0, lse[lo:hi, h]).abs())
    return out, tol, lse, lse_tol


def attend(ctx, b, q, window=0, scale=None, want_lse=True, work=None, out=None):
    heads = q.shape[1]
    work = work or paged.AttnWorkspace(ctx, heads, b.hk, b.dim)
    out = torch.full_like(q, 77.0) if out is None else out
    lse = torch.full(q.shape[:2], 55.0, device="cuda") if want_lse else None
    paged.attn_paged(ctx, b.kv, b.seqs, q, out, work, scale=scale, window=window, lse=lse)
    return out, lse


def check_attend(ctx, b, q, window=0, scale=None, want_lse=True):
    out, lse = attend(ctx, b, q, window, scale, want_lse)
    ctx.sync()
    check_result(b, q, out, lse, window, scale)
    return out


def check_result(b, q, out, lse, window=0, scale=None):
    ref, tol, rl, lt = formula(b, q, b.dim ** -0.5 if scale is None else scale, window)
    own = torch.zeros(b.n_rows, dtype=torch.bool, device="cuda")
    own[b.start[0]:b.start[-1]] = True
    assert (out[~own] == 77).all()
    err = (out[own].double() - ref[own]).abs()
    assert torch.isfinite(out[own]).all()
    worst = (err / tol[own].clamp(min=1e-30)).max().item() if err.numel() else 0.0
    assert (err <= tol[own]).all(), worst
    if lse is not None:
        assert (lse[~own] == 55).all()
        a, r, t = lse[own].double(), rl[own], lt[own]
        inf = torch.isinf(r)
        assert torch.equal(torch.isinf(a) & (a < 0), inf)
        assert ((a - r).abs()[~inf] <= t[~inf]).all()


# ---- attention ---------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 2, 128), (14, 2, 64), (4, 4, 32), (6, 2, 96), (8, 2, 256),
                                                (71, 1, 64), (128, 1, 128), (28, 4, 128)])
def test_attend_decode_and_verify_rows(ctx, dtype, heads, kv_heads, dim):
    rows = [1, 5, 1, 3, 2, 7, 1]
    lens = [1, 5, 700, 130, 129, 1025, 16]
    b = Batch(rows, lens, 16, kv_heads, dim, DT[dtype], seed=heads + dim)
    check_attend(ctx, b, b.randn(b.n_rows, heads, dim))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(12, 2, 128), (14, 2, 64), (4, 4, 32), (6, 2, 96), (4, 2, 256),
                                                (7, 1, 128), (40, 1, 64)])
@pytest.mark.parametrize("page", [16, 40])
def test_attend_chunks(ctx, dtype, heads, kv_heads, dim, page):
    rows = [300, 1, 129, 17, 64]
    lens = [300, 260, 700, 1030, 64]
    b = Batch(rows, lens, page, kv_heads, dim, DT[dtype], seed=page + dim)
    check_attend(ctx, b, b.randn(b.n_rows, heads, dim))


@pytest.mark.parametrize("page", [1, 2, 4, 5, 8, 16, 24, 64, 100, 128, 256, 1000])
@pytest.mark.parametrize("rows", [[1, 2], [90, 33]])
def test_attend_page_sizes(ctx, page, rows):
    b = Batch(rows, [777, 301], page, 2, 64, torch.float16, seed=page)
    check_attend(ctx, b, b.randn(b.n_rows, 6, 64))


@pytest.mark.parametrize("window", [1, 2, 17, 128, 129, 500, 100000])
@pytest.mark.parametrize("rows,lens", [([1, 4, 1], [900, 700, 3]), ([200, 64, 150], [900, 64, 700])])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_window(ctx, window, rows, lens, dim):
    b = Batch(rows, lens, 32, 2, dim, torch.bfloat16, seed=window)
    check_attend(ctx, b, b.randn(b.n_rows, 8, dim), window=window)


@pytest.mark.parametrize("rows,lens", [
    ([1], [1]), ([0, 1, 0, 2, 0], [0, 1, 50, 2, 7]),      # sequences without rows
    ([4, 2], [2, 0]),                                      # rows before position 0: they see nothing
    ([0, 0], [5, 0]), ([1, 1], [128, 129]), ([130], [128]), ([256], [256]), ([300, 2], [100, 2])])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_lengths_at_the_edges(ctx, rows, lens, dim):
    b = Batch(rows, lens, 16, 2, dim, torch.float16, seed=3, first=2)
    check_attend(ctx, b, b.randn(b.n_rows, 4, dim))


def test_attend_many_sequences(ctx):
    n = 1100          # more than one sequence a thread of the schedule
    rows = [(7 * i) % 3 for i in range(n)]
    lens = [1 + (i * 37) % 150 + 3 for i in range(n)]
    b = Batch(rows, lens, 16, 1, 64, torch.float16, seed=4)
    check_attend(ctx, b, b.randn(b.n_rows, 2, 64))


def test_attend_4096_sequences(ctx):
    rows, lens = [1] * 4096, [1 + i % 40 for i in range(4096)]
    b = Batch(rows, lens, 64, 1, 32, torch.float16, seed=4)
    check_attend(ctx, b, b.randn(b.n_rows, 1, 32))


@pytest.mark.parametrize("rows", [1, 7, 20, 31, 60])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_long_context_joined_from_many_parts(ctx, rows, dim):
    b = Batch([rows], [60000], 64, 2, dim, torch.float16, seed=6)
    q = b.randn(b.n_rows, 8, dim)
    first = check_attend(ctx, b, q)
    for _ in range(10):
        out, _ = attend(ctx, b, q)
        assert torch.equal(out, first)


@pytest.mark.parametrize("most", [10, 32, 200])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_many_units_a_cta(ctx, most, dim):
    """Hundreds of sequences of every small number of tiles: each CTA runs through dozens of units."""
    n = 900
    rows = [1 + (i * 13) % most for i in range(n)]
    lens = [r + (i * 101) % 900 for i, r in enumerate(rows)]
    b = Batch(rows, lens, 16, 1, dim, torch.bfloat16, seed=5)
    check_attend(ctx, b, b.randn(b.n_rows, 4, dim))


def test_attend_slots_strides_and_scale(ctx):
    b = Batch([3, 50, 1], [80, 50, 200], 16, 2, 128, torch.bfloat16, seed=8, slots=[4, 0, 2])
    packed = b.randn(b.n_rows, 8 + 4 + 8, 128)
    out = torch.full((b.n_rows, 24, 128), 77.0, device="cuda", dtype=torch.bfloat16)
    q = packed[:, 2:10]
    attend(ctx, b, q, scale=0.05, want_lse=False, out=out[:, 8:16])
    ctx.sync()
    check_result(b, q, out[:, 8:16], None, scale=0.05)
    assert (out[:, :8] == 77).all() and (out[:, 16:] == 77).all()
    # heads before rows
    qt = q.transpose(0, 1).contiguous().transpose(0, 1)
    got, _ = attend(ctx, b, qt, scale=0.05, want_lse=False)
    assert torch.equal(got, out[:, 8:16])


@pytest.mark.parametrize("rows", [6, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_attend_hidden_values_reach_nothing(ctx, rows, bad):
    """A row's result does not change when a later position's K and V are not finite."""
    b = Batch([rows, rows], [rows + 300, rows], 16, 2, 128, torch.float16, seed=9)
    q = b.randn(b.n_rows, 4, 128)
    at = rows // 2                                     # row whose own K and V go bad, in both sequences
    ref, tol, _, _ = formula(b, q, 128 ** -0.5)
    for s in range(2):
        p = b.lens[s] - rows + at
        pg = int(b.table[s, p // 16])
        b.k[pg, :, p % 16, 5] = bad
        b.v[pg, :, p % 16, 3] = bad
    out, _ = attend(ctx, b, q)
    ctx.sync()
    for s in range(2):
        lo = b.start[s]
        err = (out[lo:lo + at].double() - ref[lo:lo + at]).abs()
        assert (err <= tol[lo:lo + at]).all()
        seen = out[lo + at:lo + rows].float()
        if bad != bad:
            assert torch.isnan(seen).all()             # a NaN score spoils the rows that see it


@pytest.mark.parametrize("rows", [1, 100])
def test_attend_visible_infinite_value(ctx, rows):
    b = Batch([rows], [300], 16, 1, 64, torch.bfloat16, seed=10)
    q = b.randn(b.n_rows, 2, 64)
    pg = int(b.table[0, 1])
    b.v[pg, 0, 4, 7] = float("inf")
    out, _ = attend(ctx, b, q)
    ctx.sync()
    col = out[:rows, :, 7].float()
    assert (torch.isinf(col) & (col > 0)).all()
    assert torch.isfinite(out[:rows, :, :7]).all() and torch.isfinite(out[:rows, :, 8:]).all()


@pytest.mark.parametrize("rows", [2, 150])
def test_attend_large_scores(ctx, rows):
    """Scores of hundreds: the running maximum keeps every weight in range."""
    b = Batch([rows], [600], 16, 2, 64, torch.float16, seed=11)
    q = (b.randn(b.n_rows, 4, 64).float() * 60).half()
    check_attend(ctx, b, q)


@pytest.mark.parametrize("rows", [1, 120])
def test_attend_bad_pages_are_reported(ctx, rows):
    b = Batch([rows, rows], [400, 500], 16, 2, 64, torch.float16, seed=12)
    q = b.randn(b.n_rows, 4, 64)
    good, _ = attend(ctx, b, q)
    ctx.sync()
    for bad in (-1, b.k.shape[0], 2 ** 30):
        kept = int(b.table[0, 3])
        b.table[0, 3] = bad
        out, _ = attend(ctx, b, q)
        with pytest.raises(ALMError, match="outside its range"):
            ctx.sync()
        ctx.sync()                                     # reported once
        assert torch.equal(out[rows:2 * rows], good[rows:2 * rows])
        b.table[0, 3] = kept
    # a slot that is no row of the table, a length that the table cannot hold
    b2 = Batch([rows], [100], 16, 2, 64, torch.float16, seed=12, slots=[0])
    b2.seqs._keep[3].fill_(9)
    attend(ctx, b2, b2.randn(b2.n_rows, 4, 64))
    with pytest.raises(ALMError):
        ctx.sync()


def test_attend_is_the_same_every_time(ctx):
    b = Batch([1, 9, 1, 200], [5000, 900, 33, 1500], 16, 2, 128, torch.float16, seed=13)
    q = b.randn(b.n_rows, 12, 128)
    work = paged.AttnWorkspace(ctx, 12, 2, 128)
    first, l0 = attend(ctx, b, q, work=work)
    for _ in range(5):
        out, l1 = attend(ctx, b, q, work=work)
        assert torch.equal(out, first) and torch.equal(l1, l0)


def test_attend_high_pages(ctx):
    """Page offsets that pass 2^31 elements (and 2^32 bytes)."""
    page, dim = 128, 128
    n_pages = (1 << 31) // (page * dim) + 600
    k = torch.empty(n_pages, 1, page, dim, device="cuda", dtype=torch.float16)
    v = torch.empty_like(k)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    for rows in (2, 130):
        b = Batch([rows], [500], page, 1, dim, torch.float16, seed=2)
        at = torch.tensor([n_pages - 1, 3, n_pages - 40, n_pages - 300], device="cuda")
        k[at] = b.k[b.table[0, :4].long()]
        v[at] = b.v[b.table[0, :4].long()]
        b.table[0, :4] = at.int()
        b.k, b.v = k, v
        b.kv = paged.PagedKV(k, v)
        check_attend(ctx, b, b.randn(b.n_rows, 3, dim))


def test_attend_replayed_with_new_lengths_on_its_stream():
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c = ops.Context(0, st.cuda_stream)
        b = Batch([2, 2], [900, 20], 16, 2, 128, torch.float16, seed=14)
        q = b.randn(b.n_rows, 4, 128)
        work = paged.AttnWorkspace(c, 4, 2, 128)
        out = torch.full_like(q, 77.0)
        st.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            paged.attn_paged(c, b.kv, b.seqs, q, out, work)
        for lens in ([900, 20], [3, 17], [450, 2]):
            b.lens = lens
            b.seqs._keep[1].copy_(ints(lens))
            out.fill_(77.0)
            graph.replay()
            c.sync()
            check_result(b, q, out, None)


def test_two_captured_calls_with_their_own_work_areas():
    outs, graphs, streams, refs = [], [], [], []
    for i in range(2):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            c = ops.Context(0, st.cuda_stream)
            b = Batch([1], [30000], 64, 4, 128, torch.float16, seed=20 + i)
            q = b.randn(b.n_rows, 28, 128)
            ref, _ = attend(c, b, q)
            work, out = paged.AttnWorkspace(c, 28, 4, 128), torch.full_like(q, 77.0)
            st.synchronize()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                paged.attn_paged(c, b.kv, b.seqs, q, out, work)
            graphs.append((g, c, b, work, q))
            outs.append(out)
            refs.append(ref)
            streams.append(st)
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].zero_()
                graphs[i][0].replay()
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i][:1], refs[i][:1])


def test_context_keeps_the_callers_device_and_refuses_a_small_work_area(ctx):
    before = torch.cuda.current_device()
    b = Batch([1], [20], 16, 2, 64, torch.float16)
    q = b.randn(b.n_rows, 4, 64)
    w = paged.AttnWorkspace(ctx, 4, 2, 64)
    w.nbytes -= 4
    with pytest.raises(ALMError, match="too small"):
        paged.attn_paged(ctx, b.kv, b.seqs, q, torch.empty_like(q), w)
    assert torch.cuda.current_device() == before


# ---- norm, rotation, append ----------------------------------------------------
def table_of(n, rot, dtype, theta=10000.0):
    half = rot // 2
    ang = torch.arange(n, dtype=torch.float64, device="cuda")[:, None] * \
        theta ** (-torch.arange(half, dtype=torch.float64, device="cuda") / half)
    return torch.cat([ang.cos(), ang.sin()], 1).to(dtype)


def turned(x, w, table, pos, rot, inter, eps):
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    cs = table.double()[pos][:, None]
    c, s = cs[..., :rot // 2], cs[..., rot // 2:]
    y = x.clone()
    ia = torch.arange(0, rot, 2, device="cuda") if inter else torch.arange(rot // 2, device="cuda")
    ib = ia + (1 if inter else rot // 2)
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def near(got, ref, dtype):
    tol = torch.finfo(dtype).eps / 2 * ref.abs() + 2.0 ** -20 * ref.abs().amax(-1, keepdim=True) + 2.0 ** -25
    assert ((got.double() - ref).abs() <= tol).all()


@pytest.mark.parametrize("dtype,tdtype", [("f16", "f16"), ("f16", "f32"), ("bf16", "f32"), ("bf16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(12, 2, 128, 128), (14, 2, 64, 64), (28, 4, 128, 64), (4, 1, 32, 16),
                                                    (5, 5, 96, 96), (3, 1, 96, 48), (8, 2, 256, 256), (70, 10, 256, 64)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("norm", ["both", "none", "q", "k"])
def test_append(ctx, dtype, tdtype, heads, kv_heads, dim, rot, inter, norm):
    dt = DT[dtype]
    rows, lens = [1, 0, 5, 33, 2], [1, 9, 700, 33, 17]
    b = Batch(rows, lens, 16, kv_heads, dim, dt, seed=dim + rot, first=1)
    x = b.randn(b.n_rows, heads + 2 * kv_heads, dim) * 3
    q, k, v = x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]
    qw = (1 + b.randn(dim).float() * 0.3).to(dt) if norm in ("both", "q") else None
    kw = (1 + b.randn(dim).float() * 0.3).to(dt) if norm in ("both", "k") else None
    table = table_of(701, rot, DT[tdtype])
    k0, v0 = b.k.clone(), b.v.clone()
    out = torch.full((b.n_rows, heads, dim), 77.0, device="cuda", dtype=dt)
    paged.rope_append(ctx, b.kv, b.seqs, q, k, v, table, out, q_norm=qw, k_norm=kw, eps=1e-5, interleaved=inter)
    ctx.sync()
    touched = torch.zeros(b.k.shape[0], 16, dtype=torch.bool, device="cuda")
    for s, n in enumerate(rows):
        if n == 0:
            continue
        lo, hi = b.start[s], b.start[s + 1]
        pos = torch.arange(lens[s] - n, lens[s], device="cuda")
        near(out[lo:hi], turned(q[lo:hi], qw, table, pos, rot, inter, 1e-5), dt)
        pg = b.table[s].long()[pos // 16]
        near(b.k[pg, :, pos % 16], turned(k[lo:hi], kw, table, pos, rot, inter, 1e-5), dt)
        assert torch.equal(b.v[pg, :, pos % 16], v[lo:hi])
        touched[pg, pos % 16] = True
    assert (out[:1] == 77).all() and (out[b.start[-1]:] == 77).all()
    left = ~touched[:, None, :, None].expand_as(k0)
    for a, a0 in ((b.k, k0), (b.v, v0)):
        assert torch.equal(a[left].view(torch.int16), a0[left].view(torch.int16))


def test_append_in_place_and_other_strides(ctx):
    b = Batch([3, 4], [40, 4], 5, 2, 64, torch.float16, seed=31)
    x = b.randn(b.n_rows, 8, 64)
    table = table_of(64, 64, torch.float32)
    ref = torch.empty(b.n_rows, 4, 64, device="cuda", dtype=torch.float16)
    paged.rope_append(ctx, b.kv, b.seqs, x[:, :4], x[:, 4:6], x[:, 6:], table, ref)
    k1 = b.k.clone()
    y = x.transpose(0, 1).contiguous().transpose(0, 1)
    b.k.fill_(0)
    paged.rope_append(ctx, b.kv, b.seqs, y[:, :4], y[:, 4:6], y[:, 6:], table, y[:, :4])
    ctx.sync()
    n = b.start[-1]
    assert torch.equal(y[:n, :4], ref[:n]) and torch.equal(y[n:], x[n:])
    for s in range(2):
        pos = torch.arange(b.lens[s] - b.rows[s], b.lens[s], device="cuda")
        pg = b.table[s].long()[pos // 5]
        assert torch.equal(b.k[pg, :, pos % 5], k1[pg, :, pos % 5])


def test_append_out_of_range_rows_are_left_and_reported(ctx):
    table = table_of(50, 64, torch.float16)

    def go(b):
        x = b.randn(b.n_rows, 4, 64)
        out = torch.full((b.n_rows, 2, 64), 77.0, device="cuda", dtype=torch.float16)
        k0 = b.k.clone()
        paged.rope_append(ctx, b.kv, b.seqs, x[:, :2], x[:, 2:3], x[:, 3:], table, out)
        with pytest.raises(ALMError, match="outside its range"):
            ctx.sync()
        return out, k0
    # positions 48, 49 fit the table of 50, 50 and 51 do not
    b = Batch([4], [52], 16, 1, 64, torch.float16, seed=32)
    out, _ = go(b)
    assert (out[:2] != 77).any() and (out[2:] == 77).all()
    # negative positions
    b = Batch([3], [2], 16, 1, 64, torch.float16, seed=33)
    out, _ = go(b)
    assert (out[0] == 77).all() and (out[1:3] != 77).any()
    # pages outside the pool
    for bad in (-1, 10 ** 6):
        b = Batch([2, 1], [33, 5], 16, 1, 64, torch.float16, seed=34)
        b.table[0, 2] = bad
        out, k0 = go(b)
        assert (out[0] != 77).any() and (out[1] == 77).all() and (out[2] != 77).any()
    # a length behind the table's end
    b = Batch([1], [20], 16, 1, 64, torch.float16, seed=35)
    b.seqs._keep[1].fill_(16 * b.table.shape[1] + 1)
    out, k0 = go(b)
    assert (out == 77).all() and torch.equal(b.k.view(torch.int16), k0.view(torch.int16))


def test_append_zero_and_large_heads(ctx):
    """A zero head stays zero under the norm; values whose squares pass fp16 do not overflow."""
    b = Batch([2], [2], 16, 1, 128, torch.float16, seed=36)
    x = torch.zeros(b.n_rows, 4, 128, device="cuda", dtype=torch.float16)
    x[1] = 60000.0
    w = torch.ones(128, device="cuda", dtype=torch.float16)
    out = torch.empty(b.n_rows, 2, 128, device="cuda", dtype=torch.float16)
    table = table_of(4, 128, torch.float32)
    paged.rope_append(ctx, b.kv, b.seqs, x[:, :2], x[:, 2:3], x[:, 3:], table, out, q_norm=w, k_norm=w)
    ctx.sync()
    assert (out[0] == 0).all()
    near(out[1:2], turned(x[1:2, :2], w, table, torch.tensor([1], device="cuda"), 128, False, 1e-6), torch.float16)


def test_append_many_sequences_find_their_rows(ctx):
    n = 3000
    rows = [(i * 5) % 4 for i in range(n)]
    lens = [r + (i % 7) for i, r in enumerate(rows)]
    b = Batch(rows, lens, 16, 1, 32, torch.float16, seed=37)
    x = b.randn(b.n_rows, 3, 32)
    out = torch.full((b.n_rows, 1, 32), 77.0, device="cuda", dtype=torch.float16)
    table = table_of(16, 32, torch.float32)
    paged.rope_append(ctx, b.kv, b.seqs, x[:, :1], x[:, 1:2], x[:, 2:], table, out)
    ctx.sync()
    pos = torch.tensor([lens[s] - r + i for s, r in enumerate(rows) for i in range(r)], device="cuda")
    near(out[:b.start[-1]], turned(x[:b.start[-1], :1], None, table, pos, 32, False, 0), torch.float16)


# ---- verification --------------------------------------------------------------
def weights(l, t, mp):
    """e of one row in 64 bits (numpy)."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    top = l.max()
    if top == -np.inf:
        return np.zeros(l.size)
    with np.errstate(invalid="ignore"):
        e = np.where(l == top, 1.0, np.exp((l - top) / float(t)))
    e[l < top] = np.where(np.isinf(l[l < top]) | np.isinf(top), 0.0, e[l < top])   # left out at T = inf too
    e[e < float(mp)] = 0
    return e


def verify_ref(start, logits, draft, q, u, temp, min_p, k_max):
    """The rule, one sequence at a time."""
    n_seq = len(start) - 1
    tokens = np.full((n_seq, k_max + 1), -1, np.int64)
    n_acc = np.zeros(n_seq, np.int64)
    p_draft = np.zeros((n_seq, k_max))
    vocab = logits.shape[1]
    for s in range(n_seq):
        n = min(start[s + 1] - start[s], k_max + 1)
        if n <= 0:
            continue
        k, greedy = n - 1, not temp[s] > 0
        rows = []
        for i in range(n):
            l = logits[start[s] + i]
            if greedy:
                c = np.where(np.isnan(l), -np.inf, l)
                e = np.zeros(vocab)
                if c.max() > -np.inf:
                    e[int(np.argmax(c))] = 1
            else:
                e = weights(l, temp[s], min_p[s])
            z = e.sum()
            rows.append(e / z if z > 0 else e)
        for i in range(k):
            if 0 <= draft[s, i] < vocab:
                p_draft[s, i] = rows[i][draft[s, i]]
        acc = 0
        while acc < k:
            x = draft[s, acc]
            inside = 0 <= x < vocab
            qx = 1.0 if q is None or greedy else (float(q[s, acc, x]) if inside else 0.0)
            if inside and u[s, acc] * qx < rows[acc][x]:
                acc += 1
            else:
                break
        tokens[s, :acc] = draft[s, :acc]
        n_acc[s] = acc
        r = rows[acc].copy()
        if acc < k and not greedy:
            if q is None:
                if 0 <= draft[s, acc] < vocab:
                    r[draft[s, acc]] = 0
            else:
                r = np.maximum(r - np.nan_to_num(q[s, acc].astype(np.float64), nan=np.inf), 0)
            if not r.sum() > 0:
                r = rows[acc]
        if r.sum() > 0:
            cum = np.cumsum(r)
            hit = np.nonzero((cum > u[s, k] * cum[-1]) & (r > 0))[0]
            tokens[s, acc] = hit[0] if hit.size else np.nonzero(r > 0)[0][-1]
    return tokens, n_acc, p_draft


def run_verify(ctx, start, logits, draft, q, u, temp, min_p, want_p=True):
    n_seq, k = draft.shape
    tok = torch.full((n_seq, k + 1), 99, dtype=torch.int32, device="cuda")
    acc = torch.full((n_seq,), 99, dtype=torch.int32, device="cuda")
    pd = torch.full((n_seq, k), 9.0, device="cuda") if want_p else None
    dev = lambda a, t: None if a is None else torch.as_tensor(a, dtype=t, device="cuda")
    paged.verify(ctx, ints(list(start)), logits, dev(draft, torch.int32), dev(q, torch.float32), dev(u, torch.float64),
                 dev(temp, torch.float32), tok, acc, min_p=dev(min_p, torch.float32), p_draft=pd)
    ctx.sync()
    return tok, acc, pd


def check_verify(ctx, start, logits, draft, q, u, temp, min_p):
    tok, acc, pd = run_verify(ctx, start, logits, draft, q, u, temp, min_p)
    host = logits.float().cpu().numpy()
    t32 = np.asarray(temp, np.float32)
    mp = np.zeros(len(t32), np.float32) if min_p is None else np.asarray(min_p, np.float32)
    rt, ra, rp = verify_ref(start, host, draft, q, u, t32, mp, draft.shape[1])
    assert acc.cpu().numpy().tolist() == ra.tolist()
    assert tok.cpu().numpy().tolist() == rt.tolist()
    np.testing.assert_allclose(pd.cpu().numpy(), rp, rtol=1e-5, atol=1e-30)
    return ra


def verify_case(seed, ks, k_max, vocab, noise=0.7, peak=6.0):
    rng = np.random.default_rng(seed)
    n_seq = len(ks)
    start = np.concatenate([[0], np.cumsum([k + 1 for k in ks])])
    lg = rng.standard_normal((start[-1], vocab)) * 2
    for r in range(start[-1]):
        lg[r, rng.integers(0, vocab, 8)] += peak
    q = np.zeros((n_seq, k_max, vocab), np.float32)
    draft = np.zeros((n_seq, k_max), np.int64)
    for s in range(n_seq):
        for i in range(k_max):
            base = lg[start[s] + min(i, ks[s])]
            d = base + noise * rng.standard_normal(vocab)
            e = np.exp(d - d.max())
            q[s, i] = (e / e.sum()).astype(np.float32)
            draft[s, i] = rng.choice(vocab, p=e / e.sum())
    return rng, start, lg, draft, q, rng.random((n_seq, k_max + 1))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("ks,k_max,vocab", [([4], 4, 5000), ([0, 3, 1, 2, 0, 4], 4, 1001), ([1] * 20, 1, 37),
                                            ([31, 5], 31, 300), ([7, 0], 8, 32000), ([2, 2, 2], 2, 1), ([3], 3, 8)])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(ctx, dtype, ks, k_max, vocab, certain):
    for seed in range(4):
        rng, start, lg, draft, q, u = verify_case(seed, ks, k_max, vocab, noise=(0.0, 0.3, 0.7, 2.0)[seed])
        logits = torch.tensor(lg, device="cuda").to(DT[dtype])
        temp = np.where(np.arange(len(ks)) % 3 == 2, 0.0, (1.0, 0.8, 1.3, 0.05)[seed])
        min_p = np.where(np.arange(len(ks)) % 2 == 1, 0.1, 0.0) if seed % 2 else None
        check_verify(ctx, start, logits, draft, None if certain else q, u, temp, min_p)


def test_verify_large_vocabulary_accepts_some(ctx):
    rng, start, lg, draft, q, u = verify_case(5, [4, 4, 2, 0, 4, 3, 4, 4, 1, 4], 4, 151936, noise=0.4)
    logits = torch.tensor(lg, device="cuda").half()
    acc = check_verify(ctx, start, logits, draft, q, u, np.full(10, 1.0), None)
    assert acc.max() > 0 and acc.min() < 4


def test_verify_draws_at_the_ends(ctx):
    rng, start, lg, draft, q, u = verify_case(6, [2, 2, 2, 2], 2, 999)
    u[0], u[1], u[2], u[3] = 0.0, np.nextafter(1.0, 0.0), 1.0, [0.0, 1.0, 0.0]
    check_verify(ctx, start, torch.tensor(lg, device="cuda").float(), draft, q, u, np.ones(4), np.full(4, 0.02))


def test_verify_exact_borders(ctx):
    """Equal logits: p = 1 / n exactly for n a power of two, so u q = p and running sums equal to the goal are hit exactly."""
    vocab, n_seq = 64, 6
    lg = torch.full((n_seq * 2, vocab), -30000.0, device="cuda").half()
    lg[:, [5, 9, 33, 60]] = 1.5
    start = np.arange(n_seq + 1) * 2
    draft = np.full((n_seq, 1), 9)
    u = np.array([[0.25, 0.0], [np.nextafter(0.25, 0), 0.0], [0.25, 1 / 3], [0.0, 0.25], [0.0, 0.5], [0.0, 0.75]])
    tok, acc, pd = run_verify(ctx, start, lg, draft, None, u, np.ones(n_seq), None)
    assert acc.tolist() == [0, 1, 0, 1, 1, 1]
    # refused: 9 is left out and three remain; accepted: the running sum has to pass the goal
    assert tok.tolist() == [[5, -1], [9, 5], [33, -1], [9, 9], [9, 33], [9, 60]]
    assert (pd == 0.25).all()
    check_verify(ctx, start, lg, draft, None, u, np.ones(n_seq), None)


def test_verify_greedy_takes_the_first_of_equal_logits(ctx):
    lg = torch.zeros(6, 50000, device="cuda").bfloat16()
    lg[:, [40000, 17, 333]] = 2.0
    start, draft = [0, 3, 6], np.array([[17, 333], [333, 17]])
    tok, acc, pd = run_verify(ctx, start, lg, draft, None, np.random.rand(2, 3), [0.0, -1.0], None)
    assert acc.tolist() == [1, 0] and tok.tolist() == [[17, 17, -1], [17, -1, -1]]
    assert pd.tolist() == [[1.0, 0.0], [0.0, 1.0]]


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_verify_infinite_and_nan_logits(ctx, dtype):
    rng, start, lg, draft, q, u = verify_case(8, [2] * 6, 2, 700)
    lg[0:3, 5::7] = -np.inf
    lg[3:6, 3::5] = np.nan
    lg[6:9, [4, 90]] = np.inf
    lg[9:12] = -np.inf                       # nothing can be drawn
    lg[12:15] = np.nan
    lg[15:18, 1:] = -np.inf                  # one token only
    draft[5] = 0
    logits = torch.tensor(lg, device="cuda").to(DT[dtype])
    for temp in (1.0, 0.0):
        acc = check_verify(ctx, start, logits, draft, q, u, np.full(6, temp), None)
        assert acc[3] == 0 and acc[4] == 0


def test_verify_odd_drafts(ctx):
    """Tokens outside the vocabulary, zero and NaN draft probabilities, temperatures at the range's ends."""
    rng, start, lg, draft, q, u = verify_case(9, [3] * 8, 3, 400)
    draft[0, 0], draft[1, 1], draft[2, 2] = -1, 400, 2 ** 31 - 1
    q[3] = 0.0                               # accepted whenever p > 0
    q[4, 0] = np.nan
    temp = np.array([1, 1, 1, 1, 1, 1e-30, 1e30, np.inf])
    logits = torch.tensor(lg, device="cuda").half()
    acc = check_verify(ctx, start, logits, draft, q, u, temp, None)
    assert acc[0] == 0 and acc[1] <= 1 and acc[3] == 3 and acc[4] == 0
    check_verify(ctx, start, logits, draft, None, u, temp, np.full(8, 0.3))


def test_verify_identical_distributions_and_tiny_residuals(ctx):
    """q equal to p up to fp32 rounding: refusals are rare and their residual is rounding noise, decided in 64 bits."""
    rng = np.random.default_rng(10)
    n_seq, k, vocab = 64, 4, 3001
    start = np.arange(n_seq + 1) * (k + 1)
    lg = torch.tensor(rng.standard_normal((n_seq * (k + 1), vocab)) * 3, device="cuda").half()
    p = torch.softmax(lg.double(), -1).view(n_seq, k + 1, vocab)[:, :k]
    q = p.float().cpu().numpy()
    draft = torch.multinomial(p.reshape(-1, vocab), 1).view(n_seq, k).cpu().numpy()
    u = rng.random((n_seq, k + 1))
    u[::2, 1] = 1.0                          # at the border on purpose
    check_verify(ctx, start, lg, draft, q, u, np.ones(n_seq), None)


def test_verify_strides_and_sequences_without_rows(ctx):
    rng, start, lg, draft, q, u = verify_case(11, [2, 1, 3], 3, 333)
    wide = torch.zeros(len(lg), 400, device="cuda", dtype=torch.float16)
    wide[:, 1:334] = torch.tensor(lg, device="cuda").half()
    view = wide[:, 1:334]                    # rows that are not 16-byte aligned
    host = view.float().cpu().numpy()
    qd = torch.tensor(q, device="cuda").transpose(0, 1).contiguous().transpose(0, 1)   # step before sequence
    tok = torch.full((3, 4), 99, dtype=torch.int32, device="cuda")
    acc = torch.full((3,), 99, dtype=torch.int32, device="cuda")
    f = lambda a, t: torch.as_tensor(a, dtype=t, device="cuda")
    paged.verify(ctx, ints(list(start)), view, f(draft, torch.int32), qd, f(u, torch.float64), torch.ones(3, device="cuda"),
                 tok, acc)
    ctx.sync()
    rt, ra, _ = verify_ref(start, host, draft, q, u, np.ones(3, np.float32), np.zeros(3), 3)
    assert tok.cpu().numpy().tolist() == rt.tolist() and acc.tolist() == ra.tolist()
    # a sequence without rows between the others, and one with more rows than k_max + 1
    s2 = [0, 3, 3, 9]
    check_verify(ctx, s2, torch.tensor(lg, device="cuda").half(), draft, q, u, np.ones(3), None)


# ---- together ------------------------------------------------------------------
def test_step_on_device_append_attend_verify(ctx):
    """The operators of one verify pass in a row, captured into a graph: two
    passes over one cache, each against the formulas on the values so far."""
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c = ops.Context(0, st.cuda_stream)
        heads, hk, d, vocab = 6, 2, 64, 777
        rows, lens = [3, 1, 2], [30, 1, 130]
        b = Batch(rows, lens, 16, hk, d, torch.float16, seed=41, tail=0)
        x = b.randn(b.n_rows, heads + 2 * hk, d)
        q, k, v = x[:, :heads], x[:, heads:heads + hk], x[:, heads + hk:]
        table = table_of(256, d, torch.float32)
        w = torch.ones(d, device="cuda", dtype=torch.float16)
        qo, out = torch.empty(b.n_rows, heads, d, device="cuda", dtype=torch.float16), b.randn(b.n_rows, heads, d)
        proj = torch.randn(heads * d, vocab, device="cuda", dtype=torch.float16) * 0.3
        logits = torch.empty(b.n_rows, vocab, device="cuda", dtype=torch.float16)
        draft = torch.randint(0, vocab, (3, 2), device="cuda", dtype=torch.int32)
        u = torch.rand(3, 3, device="cuda", dtype=torch.float64)
        tok, acc = torch.empty(3, 3, device="cuda", dtype=torch.int32), torch.empty(3, device="cuda", dtype=torch.int32)
        temp = torch.tensor([1.0, 0.0, 0.7], device="cuda")
        work = paged.AttnWorkspace(c, heads, hk, d)
        start = ints(b.start)

        def step():
            paged.rope_append(c, b.kv, b.seqs, q, k, v, table, qo, q_norm=w, k_norm=w)
            paged.attn_paged(c, b.kv, b.seqs, qo, out, work)
            torch.matmul(out.view(b.n_rows, -1), proj, out=logits)
            paged.verify(c, start, logits, draft, None, u, temp, tok, acc)
        step()                                # cuBLAS takes its own memory before the capture
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            step()
        for i in range(2):
            if i:
                b.lens = [n + r for n, r in zip(b.lens, rows)]
                b.lens = [min(n, b.table.shape[1] * 16) for n in b.lens]
                # pages for the positions that were added
                used = set(b.table.flatten().tolist())
                free = iter([p for p in range(b.k.shape[0]) if p not in used])
                for s in range(3):
                    for j in range(-(-b.lens[s] // 16)):
                        if int(b.table[s, j]) < 0:
                            b.table[s, j] = next(free)
                b.seqs._keep[1].copy_(ints(b.lens))
                x.copy_(b.randn(*x.shape))
            g.replay()
            c.sync()
            for s, n in enumerate(rows):
                lo, hi = b.start[s], b.start[s + 1]
                pos = torch.arange(b.lens[s] - n, b.lens[s], device="cuda")
                near(qo[lo:hi], turned(q[lo:hi], w, table, pos, d, False, 1e-6), torch.float16)
                pg = b.table[s].long()[pos // 16]
                near(b.k[pg, :, pos % 16], turned(k[lo:hi], w, table, pos, d, False, 1e-6), torch.float16)
                assert torch.equal(b.v[pg, :, pos % 16], v[lo:hi])
            check_result(b, qo, out, None)
            rt, ra, _ = verify_ref(b.start, logits.float().cpu().numpy(), draft.cpu().numpy(), None, u.cpu().numpy(),
                                   temp.cpu().numpy(), np.zeros(3), 2)
            assert tok.cpu().numpy().tolist() == rt.tolist() and acc.tolist() == ra.tolist()


def test_operators_on_a_models_own_cache(model_dirs, golden_models):
    """A model's cache after its prefill, through DeviceKV.view and page_table:
    what rope_append writes is read back by DeviceKV.read, and attn_paged
    equals the formula on the cache's own values; without torch arrays
    (DeviceArray views of the library's memory)."""
    from androidllm_b200.ops import Context, DeviceBuffer, DeviceKV, DeviceModel
    from androidllm_b200.paged import DeviceArray
    c = Context(0)
    m = DeviceModel.from_dir(c, model_dirs["toy"])
    canon = m.canon
    h, hk, d = canon["heads"], canon["kv_heads"], canon["head_dim"]
    kv = DeviceKV(m, 64, slots=2)
    kv.set_pages(0, [3, 0])
    rng = np.random.default_rng(0)
    m.prefill(kv, rng.integers(0, canon["vocab"], 20), slot=0)
    view, n_new, length = kv.view(0), 3, 23

    def up(a, dtype):
        buf = DeviceBuffer(c, max(a.nbytes, 16))
        buf.upload(a)
        return DeviceArray(buf, a.shape, dtype)
    x = rng.standard_normal((n_new, h + 2 * hk, d)).astype(np.float16)
    q, k, v = (np.ascontiguousarray(a) for a in (x[:, :h], x[:, h:h + hk], x[:, h + hk:]))
    seqs = paged.SeqBatch(up(np.array([0, n_new], np.int32), "int32"), up(np.array([length], np.int32), "int32"),
                          kv.page_table(), n_rows=n_new)
    rope = up(m.rope, "float16")
    qo, out = up(np.zeros_like(q), "float16"), up(np.zeros_like(q), "float16")
    paged.rope_append(c, view, seqs, up(q, "float16"), up(k, "float16"), up(v, "float16"), rope, qo)
    paged.attn_paged(c, view, seqs, qo, out, paged.AttnWorkspace(c, h, hk, d))
    c.sync()
    k_all, v_all = kv.read(0, 0, length)
    r = m.rope[20:23].astype(np.float64)[:, None]
    cos, sin = r[..., :d // 2], r[..., d // 2:]

    def turn(a):
        a, b_ = a[..., :d // 2].astype(np.float64), a[..., d // 2:].astype(np.float64)
        return np.concatenate([a * cos - b_ * sin, b_ * cos + a * sin], -1)
    np.testing.assert_allclose(k_all[20:].astype(np.float64), turn(k), rtol=2.0 ** -11, atol=2.0 ** -18)
    assert np.array_equal(v_all[20:], v)
    qg = qo.buf.download(np.empty_like(q)).astype(np.float64)
    np.testing.assert_allclose(qg, turn(q), rtol=2.0 ** -11, atol=2.0 ** -18)
    got = out.buf.download(np.empty_like(q)).astype(np.float64)
    for i in range(n_new):
        for a in range(h):
            n = 21 + i
            kk, vv = (z[:n, a * hk // h].astype(np.float64) for z in (k_all, v_all))
            s = kk @ qg[i, a] / math.sqrt(d)
            w = np.exp(s - s.max())
            ref, big = w @ vv / w.sum(), w @ np.abs(vv) / w.sum()
            # the output's half step, the weights' (2^-11 of big), fp32 sums
            assert (np.abs(got[i, a] - ref) <= 2.0 ** -11 * np.abs(ref) + (2.0 ** -11 + 1e-4) * big + 1e-6).all()
    # the other slot is untouched
    k1, _ = kv.read(0, 0, 32, slot=1)
    assert not k1.any()


def test_empty_batches_do_nothing(ctx):
    k = torch.zeros(2, 1, 16, 64, device="cuda", dtype=torch.float16)
    kv, work = paged.PagedKV(k, k.clone()), paged.AttnWorkspace(ctx, 2, 1, 64)
    table = torch.zeros(1, 2, device="cuda", dtype=torch.int32)
    for n_seq in (0, 1):
        seqs = paged.SeqBatch(ints([0] * (n_seq + 1)), ints([5] * n_seq), table, n_rows=0)
        q = torch.zeros(0, 2, 64, device="cuda", dtype=torch.float16)
        one = torch.zeros(0, 1, 64, device="cuda", dtype=torch.float16)
        paged.attn_paged(ctx, kv, seqs, q, torch.empty_like(q), work)
        paged.rope_append(ctx, kv, seqs, q, one, one, table_of(4, 64, torch.float32), torch.empty_like(q))
    f = lambda *s: torch.zeros(*s, device="cuda")
    paged.verify(ctx, ints([0]), f(0, 10).half(), ints([]).view(0, 2), None, f(0, 3).double(), f(0), ints([]).view(0, 3),
                 ints([]))
    # sequences without rows: nothing accepted, nothing emitted
    tok, acc = torch.full((2, 1), 9, device="cuda", dtype=torch.int32), ints([9, 9])
    paged.verify(ctx, ints([0, 0, 0]), f(0, 10).half(), ints([]).view(2, 0), None, f(2, 1).double(), f(2), tok, acc)
    ctx.sync()
    assert tok.tolist() == [[-1], [-1]] and acc.tolist() == [0, 0] and not k.any()


def test_attend_rows_with_a_nan_query(ctx):
    """A NaN in a row's query spoils that row of that head alone."""
    for rows in (3, 100):
        b = Batch([rows], [rows + 200], 16, 2, 64, torch.float16, seed=50)
        q = b.randn(b.n_rows, 4, 64)
        ref, _ = attend(ctx, b, q)
        q[1, 2, 5] = float("nan")
        out, _ = attend(ctx, b, q)
        ctx.sync()
        assert torch.isnan(out[1, 2]).all()
        out[1, 2] = ref[1, 2]
        assert torch.equal(out, ref)


@pytest.mark.parametrize("rows", [1, 90])
def test_attend_odd_query_strides(ctx, rows):
    """Rows closer than heads, one row repeated by a stride of 0, and a tensor of one head."""
    b = Batch([rows], [rows + 60], 16, 1, 64, torch.float16, seed=51, tail=0)
    q = b.randn(1, 4, 64)
    wide = q.expand(rows, 4, 64)                       # row stride 0
    out, _ = attend(ctx, b, wide, want_lse=False, out=torch.full((rows, 4, 64), 77.0, device="cuda", dtype=q.dtype))
    ctx.sync()
    check_result(b, wide, out, None)
    one = b.randn(rows, 1, 64)
    check_attend(ctx, b, one)


def test_captured_after_a_copy_and_before_one(ctx):
    """The operators' launches overlap the previous kernel's end; copies and fills around them stay ordered."""
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        c = ops.Context(0, st.cuda_stream)
        b = Batch([4], [300], 16, 2, 64, torch.float16, seed=52, tail=0)
        src, q = b.randn(4, 8, 64), torch.zeros(4, 4, 64, device="cuda", dtype=torch.float16)
        new = torch.zeros(4, 4, 64, device="cuda", dtype=torch.float16)
        out, kept = torch.zeros_like(q), torch.zeros_like(q)
        work, table = paged.AttnWorkspace(c, 4, 2, 64), table_of(300, 64, torch.float32)

        def step():
            q.copy_(src[:, :4])
            new.copy_(src[:, 4:])
            paged.rope_append(c, b.kv, b.seqs, q, new[:, :2], new[:, 2:], table, q)
            paged.attn_paged(c, b.kv, b.seqs, q, out, work)
            kept.copy_(out)
            q.zero_()
            out.zero_()
        st.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            step()
        for _ in range(3):
            src.copy_(b.randn(4, 8, 64))
            g.replay()
            c.sync()
            pos = torch.arange(296, 300, device="cuda")
            turned_q = turned(src[:, :4], None, table, pos, 64, False, 0).half()
            ref, tol, _, _ = formula(b, turned_q, 64 ** -0.5)
            # one more half step a query value: the rotation's own rounding may fall to the other side
            slack = 2.0 ** -10 * 64 ** -0.5 * 64 * 4
            assert ((kept.double() - ref).abs() <= tol + slack * 4).all() and not out.any() and not q.any()
            step()
            c.sync()


def test_two_contexts_at_once():
    """Calls of two contexts on two streams, without waiting in between."""
    todo = []
    for i in range(2):
        st = torch.cuda.Stream()
        with torch.cuda.stream(st):
            c = ops.Context(0, st.cuda_stream)
            b = Batch([7, 300], [5000, 700], 16, 2, 128, torch.bfloat16, seed=60 + i)
            q = b.randn(b.n_rows, 14, 128)
            ref, _ = attend(c, b, q)
            todo.append((st, c, b, q, paged.AttnWorkspace(c, 14, 2, 128), ref))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for i, (st, c, b, q, work, _) in enumerate(todo):
            with torch.cuda.stream(st):
                outs[i].append(attend(c, b, q, work=work)[0])
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, todo[i][5]) for o in outs[i])


def test_cuda_array_interface_arrays(ctx):
    class Cai:
        def __init__(self, t):
            self.t = t
            self.shape = tuple(t.shape)
            kind = {torch.float16: "<f2", torch.int32: "<i4", torch.float32: "<f4"}[t.dtype]
            size = t.element_size()
            self.__cuda_array_interface__ = {"data": (t.data_ptr(), False), "shape": self.shape, "typestr": kind,
                                             "strides": tuple(s * size for s in t.stride()), "version": 3}
    b = Batch([2], [40], 16, 2, 64, torch.float16, seed=53)
    q = b.randn(b.n_rows, 4, 64)
    ref, _ = attend(ctx, b, q)
    kv = paged.PagedKV(Cai(b.k), Cai(b.v))
    seqs = paged.SeqBatch(Cai(ints(b.start)), Cai(ints(b.lens)), Cai(b.table), n_rows=b.n_rows, max_rows=2)
    out = torch.full_like(q, 77.0)
    paged.attn_paged(ctx, kv, seqs, Cai(q), Cai(out), paged.AttnWorkspace(ctx, 4, 2, 64))
    ctx.sync()
    assert torch.equal(out, ref)


def test_row_starts_that_do_not_rise_are_harmless(ctx):
    """Rows claimed by no sequence or by a falling start are not computed; nothing is read out of range."""
    b = Batch([3, 2], [30, 20], 16, 1, 64, torch.float16, seed=54)
    q = b.randn(b.n_rows, 2, 64)
    for start in ([0, 3, 1], [5, 0, 2], [-4, 3, 5], [0, 3, 10 ** 9]):
        b.seqs._keep[0].copy_(ints(start))
        attend(ctx, b, q)
        x = b.randn(b.n_rows, 4, 64)
        paged.rope_append(ctx, b.kv, b.seqs, x[:, :2], x[:, 2:3], x[:, 3:], table_of(64, 64, torch.float32),
                          torch.empty(b.n_rows, 2, 64, device="cuda", dtype=torch.float16))
        try:
            ctx.sync()
        except ALMError:
            pass


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("n_seq", [5, 40])          # CTAs fewer and more than SMs
def test_verify_infinities_at_every_temperature(ctx, dtype, n_seq):
    rng, start, lg, draft, q, u = verify_case(70, [2] * n_seq, 2, 600)
    lg[3:6, 5::7] = -np.inf
    lg[6:9, [4, 90]] = np.inf
    lg[7, 91] = np.nan
    lg[9:12] = -np.inf
    u[3] = 0.0
    logits = torch.tensor(lg, device="cuda").to(DT[dtype])
    for temp in (1e-36, 1e-3, 1.0, 1e33, np.inf):
        for min_p in (0.0, 0.3, 1.0):
            check_verify(ctx, start, logits, draft, q, u, np.full(n_seq, temp), np.full(n_seq, min_p))


@pytest.mark.parametrize("noise", [1e-6, 1e-5, 1e-4, 1e-3])
def test_verify_drafts_close_to_the_model(ctx, noise):
    """q off p by factors of 1 +- noise: many entries at the residual's border, then some, then few."""
    rng = np.random.default_rng(71)
    n_seq, k, vocab = 24, 2, 20011
    start = np.arange(n_seq + 1) * (k + 1)
    lg = torch.tensor(rng.standard_normal((n_seq * (k + 1), vocab)) * 2, device="cuda").half()
    p = torch.softmax(lg.double(), -1).view(n_seq, k + 1, vocab)[:, :k].cpu().numpy()
    q = (p * (1 + noise * rng.standard_normal(p.shape))).astype(np.float32)
    draft = rng.integers(0, vocab, (n_seq, k))
    u = rng.random((n_seq, k + 1))
    u[:, :k] = 1.0 + 1e-2                    # refuse at once: the residual decides
    check_verify(ctx, start, lg, draft, q, u, np.ones(n_seq), None)


def test_one_work_area_for_several_shapes(ctx):
    """Calls in turn with other head dimensions, row counts and kernels through one area."""
    work = paged.AttnWorkspace(ctx, 16, 2, 128)
    cases = []
    for i, (rows, n_kv, heads, hk, dim) in enumerate([(1, 700, 14, 2, 128), (1, 900, 14, 2, 64), (40, 900, 12, 2, 64),
                                                      (1, 3000, 4, 1, 32), (4, 2000, 14, 2, 128), (1, 333, 8, 2, 96)]):
        b = Batch([rows] * 3, [n_kv, n_kv // 2 + rows, rows], 16, hk, dim, torch.float16, seed=80 + i)
        q = b.randn(b.n_rows, heads, dim)
        cases.append((b, q, attend(ctx, b, q)[0]))
    for _ in range(3):
        for b, q, ref in cases:
            out, _ = attend(ctx, b, q, work=work)
            ctx.sync()
            assert torch.equal(out, ref)


@pytest.mark.parametrize("table", [64, 400])
def test_decode_rows_joined_either_way(ctx, table):
    """One long sequence: a small page table has the last CTA join, a large one the kernel."""
    b = Batch([1], [1000], 16, 2, 128, torch.bfloat16, seed=90)
    wide = torch.zeros(1, table, device="cuda", dtype=torch.int32)
    wide[:, :b.table.shape[1]] = b.table[:1]
    b.seqs = paged.SeqBatch(ints(b.start), ints(b.lens), wide, n_rows=b.n_rows, max_rows=1)
    q = b.randn(b.n_rows, 8, 128)
    check_attend(ctx, b, q)


# ---- values that are not finite, beside units that follow ----------------------
def not_finite_at(b, s, pos, value, col=None):
    """Makes V of sequence s at this position not finite (every column, or one)."""
    page = int(b.table[b.slot[s], pos // b.page])
    b.v[page, :, pos % b.page, slice(None) if col is None else col] = value


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("most", [16, 30])
def test_attend_hidden_nan_in_many_short_units(ctx, dim, most):
    """Each CTA runs through units whose every row has a NaN just before its
    window: the rows recomputed at one unit's end are not lost to the next."""
    n = 700
    rows = [most - i % 4 for i in range(n)]
    lens = [r + 20 + (i * 29) % 90 for i, r in enumerate(rows)]
    b = Batch(rows, lens, 16, 1, dim, torch.float16, seed=41)
    for s in range(n):
        not_finite_at(b, s, lens[s] - rows[s] - 6, float("nan"))
    q = b.randn(b.n_rows, 1, dim)
    for _ in range(3):
        check_attend(ctx, b, q, window=6)


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 200, 1024, 60])
@pytest.mark.parametrize("rows,lens", [([6], [3]), ([6, 1, 40], [2, 900, 9]), ([300, 5], [100, 700])])
@pytest.mark.parametrize("dim", [64, 96])
def test_attend_windows_beyond_every_position(ctx, window, rows, lens, dim):
    """A window near 2^31 hides nothing, also where rows lie before position 0."""
    b = Batch(rows, lens, 16, 2, dim, torch.float16, seed=42, first=1)
    q = b.randn(b.n_rows, 8, dim)
    out = check_attend(ctx, b, q, window=window)
    if window > 1000:
        plain, _ = attend(ctx, b, q)
        assert torch.equal(out, plain)


@pytest.mark.parametrize("rows", [1, 7, 120])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_attend_length_beyond_the_table_is_reported(ctx, rows, dim):
    """A sequence longer than its row of the table: its rows see nothing, and the next sync says so."""
    b = Batch([rows, rows], [400, 500], 16, 2, dim, torch.float16, seed=43)
    b.table[0] = b.table[0, 0]                       # every entry a page of the pool
    q = b.randn(b.n_rows, 4, dim)
    good, good_lse = attend(ctx, b, q)
    ctx.sync()
    for n in (b.table.shape[1] * 16 + 1, 2 ** 31 - 1):
        b.seqs._keep[1].copy_(ints([n, 500]))
        out, lse = attend(ctx, b, q)
        with pytest.raises(ALMError, match="outside its range"):
            ctx.sync()
        ctx.sync()                                   # reported once
        assert (out[:rows] == 0).all() and (lse[:rows] == -math.inf).all()
        assert torch.equal(out[rows:], good[rows:]) and torch.equal(lse[rows:], good_lse[rows:])
    b.seqs._keep[1].copy_(ints([b.table.shape[1] * 16, 500]))
    attend(ctx, b, q)
    ctx.sync()                                       # the last position there is


def check_not_finite(ctx, b, q, marks, window=0, times=1):
    """Rows with infinities and NaN in V at marks = (sequence, position, column,
    value): a row that sees one has it in that column (opposite infinities: NaN),
    everything else is the formula's."""
    for s, pos, col, value in marks:
        not_finite_at(b, s, pos, value, col)
    ref, tol, _, _ = formula(b, q, b.dim ** -0.5, window)
    for s, pos, col, value in marks:
        for r in range(b.rows[s]):
            p = b.lens[s] - b.rows[s] + r
            if pos <= p and not (window and pos <= p - window):
                ref[b.start[s] + r, :, col] += value
    own = slice(b.start[0], b.start[-1])
    ref, tol = ref[own], tol[own]
    some = torch.isfinite(ref)
    for _ in range(times):
        out, lse = attend(ctx, b, q, window)
        ctx.sync()                                   # no wait ran out
        got = out[own].double()
        assert torch.equal(torch.isnan(got), torch.isnan(ref))
        assert torch.equal(got[~some & ~torch.isnan(ref)], ref[~some & ~torch.isnan(ref)])
        assert ((got - ref).abs()[some] <= tol[some]).all()
        assert torch.isfinite(lse[own]).all()
        assert (out[b.start[-1]:] == 77).all()


INF, NAN = float("inf"), float("nan")


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 7, 28, 300])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_attend_infinities_over_a_long_context(ctx, dtype, rows, dim):
    n = 30000 if dim in (64, 128) else 6000
    b = Batch([rows, 2], [n + rows, 500], 16, 1, dim, DT[dtype], seed=45)
    marks = [(0, n // 6, 7, INF), (0, n // 6 + 1, 8, -INF), (0, 3, 9, INF), (0, n - 9, 9, -INF), (0, n // 2, 31, NAN),
             (0, n + rows // 2, 11, NAN), (0, n + rows // 2, 12, INF), (1, 450, 1, INF), (1, 499, 2, -INF)]
    check_not_finite(ctx, b, b.randn(b.n_rows, 4, dim), marks, times=2)


@pytest.mark.parametrize("window", [1, 40, 200, 1000])
@pytest.mark.parametrize("rows", [[3, 7, 1], [70, 30, 300]])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_attend_infinities_at_the_window_border(ctx, window, rows, dim):
    """Values that some rows of a block see and others do not, on both sides."""
    lens = [r + n for r, n in zip(rows, (2000, 90, 700))]
    b = Batch(rows, lens, 32, 2, dim, torch.float16, seed=46)
    marks = []
    for s in range(3):
        for i, (back, value) in enumerate([(0, NAN), (rows[s] // 2, INF), (rows[s] + 1, -INF), (window, NAN),
                                           (window + rows[s] // 2, INF), (window + rows[s], -INF), (1, -INF)]):
            if 0 <= lens[s] - 1 - back:
                marks.append((s, lens[s] - 1 - back, 5 * i + s, value))
    check_not_finite(ctx, b, b.randn(b.n_rows, 6, dim), marks, window)


@pytest.mark.parametrize("rows", [1, 20, 60])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_infinity_of_a_tiny_weight(ctx, rows, dim):
    """The weight of a visible infinity is never zero, also below what 16 or 32 bits hold."""
    n = 40000
    b = Batch([rows], [n], 16, 1, dim, torch.float16, seed=47)
    q = b.randn(b.n_rows, 2, dim).abs() + 1
    # weights of less than 2^-126 before position 12000
    pages = b.table[0, :750].long()
    b.k[pages] = -abs(b.k[pages]) - 8
    check_not_finite(ctx, b, q, [(0, 100, 3, INF), (0, 11000, 4, -INF), (0, n - 1, 5, INF)])


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("rows", [10, 50, 90])
def test_attend_not_finite_in_every_unit(ctx, dim, rows):
    """Many sequences, each with values that only some of its rows see: every unit is made twice."""
    n = 300
    b = Batch([rows - i % 3 for i in range(n)], [rows + (i * 37) % 400 for i in range(n)], 16, 1, dim, torch.bfloat16, seed=48)
    marks = [(s, b.lens[s] - 1 - s % rows, s % 32, (INF, -INF, NAN)[s % 3]) for s in range(n)]
    check_not_finite(ctx, b, b.randn(b.n_rows, 3, dim), marks, times=2)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("rows,heads,dim", [([1, 3, 1], 4, 64), ([5, 1, 2], 12, 96), ([200, 90, 1], 4, 64),
                                            ([40, 33, 2], 4, 128)])
@pytest.mark.parametrize("scale", [1e7, 1e9, 1e30])
def test_attend_scales_that_leave_one_weight(ctx, dtype, rows, heads, dim, scale):
    """Whole-number scores times a large scale: a row is the mean of the V of its
    largest scores.  Scores and weights (0 or 1) are exact, so the output is off by
    its own half step, a quotient and a few sums; lse by three roundings of itself."""
    lens = [r + n for r, n in zip(rows, (0, 700, 2))]
    b = Batch(rows, lens, 16, 2, dim, DT[dtype], seed=44)
    b.k.copy_(torch.randint(-3, 4, b.k.shape, generator=b.gen, device="cuda"))
    q = torch.randint(-3, 4, (b.n_rows, heads, dim), generator=b.gen, device="cuda").to(DT[dtype])
    out, lse = attend(ctx, b, q, scale=scale)
    ctx.sync()
    for s in range(3):
        k, v = b.cached(s)
        pos = torch.arange(lens[s] - rows[s], lens[s], device="cuda")
        hidden = torch.arange(lens[s], device="cuda")[None] > pos[:, None]
        for h in range(heads):
            kh, vh = k[h // (heads // 2)], v[h // (heads // 2)]
            sc = (q[b.start[s]:b.start[s + 1], h].double() @ kh.T).masked_fill(hidden, -math.inf)
            top = sc.amax(1, keepdim=True)
            w = (sc == top).double()
            ref, big = (w @ vh) / w.sum(1, keepdim=True), (w @ vh.abs()) / w.sum(1, keepdim=True)
            got = out[b.start[s]:b.start[s + 1], h].double()
            tol = torch.finfo(DT[dtype]).eps / 2 * ref.abs() + 2.0 ** -20 * big + 2.0 ** -25
            assert ((got - ref).abs() <= tol).all()
            # (the scale is used in 32 bits, times log2 e and back)
            rl = top[:, 0] * float(np.float32(scale)) + torch.log(w.sum(1))
            assert ((lse[b.start[s]:b.start[s + 1], h].double() - rl).abs() <= 2.0 ** -20 * rl.abs() + 2.0 ** -20).all()


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_attend_is_the_same_after_large_scores(ctx, rows):
    """What an earlier call left on chip (here: large scores) changes no bit of a result."""
    b = Batch([rows, rows], [2000, 300], 16, 2, 128, torch.float16, seed=49)
    q = b.randn(b.n_rows, 14, 128)                   # 7 heads: two of 128 rows stay unused
    first, first_lse = attend(ctx, b, q)
    for scale in (1e9, 0.05, 1e30):
        attend(ctx, b, (q.float() * 300).half(), scale=scale)
        out, lse = attend(ctx, b, q)
        assert torch.equal(out, first) and torch.equal(lse, first_lse)
    ctx.sync()


def test_verify_border_in_the_largest_vocabulary(ctx):
    """2^24 tokens of one probability but one.  Added one at a time in 32 bits a
    lane's 65536 weights of 0.998 fall short by 49% of a step each behind 2^15: by
    1e-3 of the sum.  Draws closer to p than that are still decided right."""
    vocab, k = 1 << 24, 15
    logits = torch.zeros(k + 1, vocab, device="cuda", dtype=torch.float16)
    logits[:, 5] = 1.0
    c = 255.49 / 256
    temp = np.float32(-1.0 / math.log(c))
    c = math.exp(-1.0 / float(temp))
    z = 1.0 + (vocab - 1) * c
    n_seq = 9                                        # the other sequences have no rows
    start = [0] + [k + 1] * n_seq
    draft = np.full((n_seq, k), 12345)
    for off, want in ((1 + 3e-4, 0), (1 - 3e-4, k), (1 + 1e-9, 0), (1 - 1e-9, k)):
        u = np.full((n_seq, k + 1), c / z * off)
        u[:, k] = 0.37
        tok, acc, pd = run_verify(ctx, start, logits, draft, None, u, np.full(n_seq, temp), np.full(n_seq, 1e-3))
        assert acc.tolist() == [want] + [0] * (n_seq - 1)
        # the draw: after a refusal without the drafted token's mass
        if want == k:
            at = 0.37 * z
            first = int((at - 1.0) // c) + 1         # token 5 weighs 1, those before it c each
        else:
            at = 0.37 * (z - c)
            first = int((at - 1.0) // c) + 2
        assert tok[0, want].item() == first and tok[0, :want].tolist() == [12345] * want
        np.testing.assert_allclose(pd[0].cpu().numpy(), c / z, rtol=1e-4 + 5e-7 * 8192)


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_verify_denormal_temperatures(ctx, dtype):
    """All mass on the largest logits, also where 1 / T leaves 32 bits."""
    rng, start, lg, draft, q, u = verify_case(72, [2] * 6, 2, 600)
    lg[3:6, 5::7] = -np.inf
    lg[9:12] = -np.inf
    lg = lg.astype(np.float16).astype(np.float64)
    draft[0], draft[2] = lg[start[0]:start[0] + 2].argmax(1), lg[start[2]:start[2] + 2].argmax(1)
    for temp in (1e-37, 1e-39, 1e-42, 1e-45):
        for min_p in (0.0, 0.3, 1.0):
            check_verify(ctx, start, torch.tensor(lg, device="cuda").to(DT[dtype]), draft, q, u, np.full(6, temp),
                         np.full(6, min_p))


def test_attend_refuses_q_as_its_output(ctx):
    b = Batch([3], [20], 16, 2, 64, torch.float16, seed=50)
    q = b.randn(b.n_rows, 4, 64)
    kept = q.clone()
    with pytest.raises(ALMError, match="must not be q_dev"):
        attend(ctx, b, q, out=q)
    ctx.sync()
    assert torch.equal(q, kept)
