"""Attention over the 8-bit cache, decoding rows and chunks of new rows, against plain 64-bit arithmetic."""
import math

import pytest
import torch

import plain_q8

BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    from cbis_b200.kernels import ops as o
    return o


def make(ops, dtype, H, G, hd, ps, ctx, rows, seed, spread=1.0, extra=()):
    """Requests of ``ctx`` tokens whose last ``rows`` are queries; the pages' free slots hold codes 77 with scale NaN."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-c // ps) for c in ctx]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(ctx), max(need) + 1), -1, dtype=torch.int32)
    codes = [torch.full((pages, G, ps, hd), 77, dtype=torch.int8) for _ in "kv"]
    scales = [torch.full((pages, G, ps), math.nan) for _ in "kv"]
    held = [[], []]
    at = 0
    for r, c in enumerate(ctx):
        table[r, :need[r]] = order[at:at + need[r]].to(torch.int32)
        at += need[r]
        for x in range(2):
            values = torch.randn(c, G, hd, generator=g) * spread
            code, scale = plain_q8.quantise(values)
            p = torch.arange(c)
            page = table[r, p // ps].long()
            codes[x][page, :, p % ps] = code.to(torch.int8)
            scales[x][page, :, p % ps] = scale
            held[x].append(code * scale.double()[..., None])
    q = torch.randn(sum(rows), H * hd, generator=g).to(dtype)
    positions = torch.tensor([c - n + i for c, n in zip(ctx, rows) for i in range(n)], dtype=torch.int32)
    seq = torch.tensor([r for r, n in enumerate(rows) for _ in range(n)], dtype=torch.int32)
    cu = torch.tensor([sum(rows[:r]) for r in range(len(rows) + 1)], dtype=torch.int32)
    return dict(k=ops.Q8Pages(codes[0].cuda(), scales[0].cuda()), v=ops.Q8Pages(codes[1].cuda(), scales[1].cuda()), held=held, table=table,
                q=q, positions=positions, seq=seq, cu=cu, ctx=ctx, rows=rows, H=H, G=G, hd=hd, ps=ps, dtype=dtype)


def check(c, out, scale, window=0, keep=0, rows=None, factor=1.0, **extra):
    """``extra``: slopes, rates, sinks (per head), cap, temp."""
    H, G, hd = c["H"], c["G"], c["hd"]
    out = out.double().cpu()
    for r in range(len(c["positions"])) if rows is None else rows:
        s, p = int(c["seq"][r]), int(c["positions"][r])
        keys = plain_q8.seen_keys(p, window, keep)
        for h in range(H):
            one = {n: (None if extra.get(n) is None else float(extra[n][h])) for n in ("slope", "rate", "sink")}
            ref, weighted, size = plain_q8.attend(c["q"][r, h * hd:(h + 1) * hd].double(), c["held"][0][s][:, h // (H // G)],
                                                  c["held"][1][s][:, h // (H // G)], p, keys, scale, one["slope"] or 0.0, one["rate"],
                                                  one["sink"], extra.get("cap", 0.0), extra.get("temp"))
            tol = factor * plain_q8.tolerance(c["dtype"], ref, weighted, size, hd, len(keys))
            off = (out[r, h * hd:(h + 1) * hd] - ref).abs()
            assert (off <= tol).all(), (r, h, (off / tol).max().item())


def scratch(ops, rows, most, n_seg, c, ctx=None):
    floats, counters = ops.attention_q8_scratch(rows, most, n_seg, c["H"], c["G"], c["hd"], ctx or max(c["ctx"]), c["dtype"])
    return torch.full((floats,), math.nan, device="cuda"), torch.zeros(counters, dtype=torch.int32, device="cuda")


def decode(ops, c, window=0, max_context=None, q=None, k_off=-1, v_off=-1, slots=None, out=None, seq=None, buffers=None, **kw):
    q = c["q"].cuda() if q is None else q
    seq = c["seq"] if seq is None else seq
    out = torch.full((q.shape[0], c["H"] * c["hd"]), math.nan, dtype=c["dtype"], device="cuda") if out is None else out
    buf = buffers or scratch(ops, q.shape[0], 1, 0, c, max_context)
    ops.paged_decode_q8(q, k_off, v_off, c["k"], c["v"], c["table"].cuda(), seq.cuda(), c["positions"].cuda(), slots, out, *buf, c["H"], c["G"],
                        c["hd"], c["ps"], c["hd"] ** -0.5, window, max_context or max(c["ctx"]), **kw)
    assert int(buf[1].abs().sum()) == 0      # the counters are left as they were
    return out


CTX = [1, 2, 15, 16, 17, 129, 700, 64]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps,window", [
    (3, 3, 32, 16, 0), (2, 1, 16, 8, 0), (5, 5, 64, 16, 0), (4, 4, 128, 16, 0), (2, 2, 80, 4, 0), (2, 1, 256, 32, 0), (2, 1, 144, 16, 0), (8, 1, 64, 16, 0),
    (12, 1, 128, 16, 0), (20, 1, 32, 16, 0), (40, 1, 64, 64, 0), (36, 1, 128, 3, 0), (10, 2, 96, 16, 33), (4, 2, 128, 16, -48), (2, 2, 64, 5, 7), (17, 1, 256, 16, 100)])
def test_decode(ops, dtype, H, G, hd, ps, window):
    c = make(ops, dtype, H, G, hd, ps, CTX, [1] * len(CTX), seed=hd + ps + H)
    check(c, decode(ops, c, window), hd ** -0.5, window)


@pytest.mark.gpu
@pytest.mark.parametrize("max_context", [700, 32, 32768])
def test_decode_is_the_same_however_the_grid_is_sized(ops, max_context):
    """``max_context`` sizes the grid (a captured step names the bound of its class): one block or many, the rows are whole."""
    for dtype in (BF, F32):
        c = make(ops, dtype, 4, 2, 64, 16, CTX, [1] * len(CTX), seed=1)
        check(c, decode(ops, c, max_context=max_context), 1 / 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_decode_stores_the_current_token(ops, dtype):
    """The key and value of the current token come from the projections' columns; a padding row at the end stores nothing."""
    H, G, hd, ps = 6, 2, 64, 16
    c = make(ops, dtype, H, G, hd, ps, CTX, [1] * len(CTX), seed=2)
    S, wide, dq = len(CTX), G * hd, H * hd
    qkv = torch.zeros(S + 1, dq + 2 * wide + 8, dtype=dtype)
    qkv[:S, :dq] = c["q"]
    qkv[:, dq:dq + 2 * wide] = torch.randn(S + 1, 2 * wide, generator=torch.Generator().manual_seed(9)).to(dtype)
    slots = torch.full((S + 1,), -1, dtype=torch.int32)
    before = [c["k"].codes.clone(), c["v"].codes.clone()]
    for r, n in enumerate(CTX):
        slots[r] = int(c["table"][r, (n - 1) // ps]) * ps + (n - 1) % ps
        for x, off in ((0, dq), (1, dq + wide)):
            code, scale = plain_q8.quantise(qkv[r, off:off + wide].view(G, hd))
            c["held"][x][r][n - 1] = code * scale.double()[:, None]
            before[x][int(slots[r]) // ps, :, int(slots[r]) % ps] = code.to(torch.int8).cuda()
    c["positions"] = torch.cat([c["positions"], torch.tensor([0], dtype=torch.int32)])
    seq = torch.cat([c["seq"], torch.tensor([-1], dtype=torch.int32)])
    out = decode(ops, c, q=qkv.cuda()[:, :dq + 2 * wide], k_off=dq, v_off=dq + wide, slots=slots.cuda(), seq=seq)
    assert torch.all(out[S] == 0)
    c["positions"] = c["positions"][:S]
    check(c, out, 1 / 8, rows=range(S))
    assert torch.equal(c["k"].codes, before[0]) and torch.equal(c["v"].codes, before[1])
    for r, n in enumerate(CTX):
        code, scale = plain_q8.quantise(qkv[r, dq:dq + wide].view(G, hd))
        assert torch.equal(c["k"].scales[int(slots[r]) // ps, :, int(slots[r]) % ps].cpu(), scale)


EXTRAS = [dict(cap=5.0), dict(window=40, keep=5), dict(window=33, keep=40), dict(sinks=True), dict(slopes=True), dict(slopes=True, rates=True, sinks=True),
          dict(q_temp=(0.3, 20)), dict(window=-64, keep=17, cap=3.0, sinks=True, slopes=True, q_temp=(0.1, 7))]


def numbers(kw, H):
    kw, told = dict(kw), {}
    g = torch.Generator().manual_seed(H)
    for name, one in (("sinks", "sink"), ("slopes", "slope"), ("rates", "rate")):
        if kw.get(name):
            kw[name] = torch.rand(H, generator=g) * (0.1 if name == "slopes" else 1.0)
            told[one] = kw[name].tolist()
            kw[name] = kw[name].cuda()
    window, keep = kw.pop("window", 0), kw.get("keep", 0)
    if "q_temp" in kw:
        told["temp"] = kw["q_temp"]
    if "cap" in kw:
        told["cap"] = kw["cap"]
    return kw, told, window, keep


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps", [(3, 3, 64, 16), (10, 2, 128, 16), (4, 1, 48, 6)])
@pytest.mark.parametrize("kw", EXTRAS)
def test_decode_extras(ops, dtype, H, G, hd, ps, kw):
    kw, told, window, keep = numbers(kw, H)
    c = make(ops, dtype, H, G, hd, ps, [1, 37, 300, 170], [1] * 4, seed=hd)
    check(c, decode(ops, c, window, **kw), hd ** -0.5, window, keep, **told)


def prefill(ops, c, window=0, work=False, seg0=0, out=None, max_context=None, **kw):
    n, rows = len(c["rows"]) - seg0, sum(c["rows"][seg0:])
    row0 = sum(c["rows"][:seg0])
    out = torch.full(c["q"].shape, 7.5, dtype=c["dtype"], device="cuda") if out is None else out
    buf = scratch(ops, rows, max(c["rows"]), n, c, max_context)
    pages = tuple(torch.full(c["k"].codes.shape, math.nan, dtype=c["dtype"], device="cuda") for _ in "kv") if work else None
    takes = ops.prefill_q8_reads_back
    if work:        # wherever there is a kernel over pages read back, whichever is the faster one
        ops.prefill_q8_reads_back = lambda rows, most, n_seg, *rest: takes(10 ** 9, most, n_seg, *rest) or takes(rows, 10 ** 9, n_seg, *rest)
    start = torch.tensor([a - b for a, b in zip(c["ctx"], c["rows"])], dtype=torch.int32).cuda()
    ops.paged_prefill_q8(c["q"].cuda(), c["k"], c["v"], c["table"].cuda(), c["cu"].cuda(), start, torch.tensor(c["ctx"], dtype=torch.int32).cuda(),
                         c["positions"].cuda(), out, seg0, n, row0, rows, max(c["rows"]), c["H"], c["G"], c["hd"], c["ps"], c["hd"] ** -0.5, window,
                         max_context or max(c["ctx"]), *buf, pages, **kw)
    ops.prefill_q8_reads_back = takes
    assert int(buf[1].abs().sum()) == 0
    return out


def test_which_kernel_takes_a_chunk():
    from cbis_b200.kernels import ops
    small = dict(n_seg=1, n_head=16, n_kv_head=16, head_dim=128, page_size=16, dtype=BF)
    reads = lambda rows, **kw: ops.prefill_q8_reads_back(rows, rows, **{**small, **kw})      # noqa: E731
    assert not reads(32) and reads(256) and not reads(256, head_dim=96) and not reads(256, page_size=24) and not reads(256, q_temp=(0.1, 5))
    assert not reads(256, slopes=1, rates=1) and reads(256, sinks=1) and reads(256, cap=3.0, keep=2)
    assert not reads(4096, dtype=F32) and reads(70000, dtype=F32) and not reads(70000, dtype=F32, sinks=1)      # (more row tiles than are counted)
    assert not ops.prefill_q8_takes(70000, 70000, **{**small, "dtype": F32}, sinks=1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps,window", [
    (3, 3, 32, 16, 0), (2, 1, 16, 8, 0), (4, 4, 128, 16, 0), (8, 1, 64, 16, 0), (5, 1, 80, 4, 0), (2, 1, 256, 32, 0), (10, 2, 96, 3, 33), (4, 2, 128, 16, -48),
    (40, 1, 32, 16, 0)])
def test_chunks(ops, dtype, H, G, hd, ps, window):
    """Rows of requests side by side, cut anywhere: one row, an empty request, a chunk from position 0."""
    c = make(ops, dtype, H, G, hd, ps, [1, 40, 300, 33, 29], [1, 7, 3, 0, 29], seed=hd + H)
    check(c, prefill(ops, c, window), hd ** -0.5, window)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("kw", EXTRAS)
def test_chunk_extras(ops, dtype, kw):
    kw, told, window, keep = numbers(kw, 6)
    c = make(ops, dtype, 6, 3, 64, 16, [5, 150, 260], [5, 9, 20], seed=4)
    check(c, prefill(ops, c, window, **kw), 1 / 8, window, keep, **told)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps,window", [(2, 2, 64, 16, 0), (4, 2, 128, 32, 0), (2, 1, 32, 8, 0), (2, 2, 80, 16, 50), (2, 1, 128, 16, -64), (2, 2, 64, 64, 70)])
def test_long_chunks_read_back(ops, dtype, H, G, hd, ps, window):
    """Chunks of many rows; the pages that the values are read back into hold NaN before."""
    c = make(ops, dtype, H, G, hd, ps, [190, 300, 77], [130, 90, 77], seed=hd)
    rows = list(range(0, 297, 13)) + [129, 130, 219, 220, 296]
    check(c, prefill(ops, c, window, work=True), hd ** -0.5, window, rows=rows)


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_a_key_that_is_not_finite_in_a_long_chunk(ops, hd):
    """The same over pages read back: to every row that sees it, and to no other."""
    for x in "kv":
        c = make(ops, BF, 4, 2, hd, 16, [300, 260], [150, 140], seed=9)
        c[x].scales[int(c["table"][0, 200 // 16]), 1, 200 % 16] = math.nan
        out = prefill(ops, c, work=True).cpu().view(290, 4, hd)
        for r in range(290):
            hit = r < 150 and 150 + r >= 200
            assert torch.isnan(out[r, 2:]).all().item() == hit and torch.isfinite(out[r, :2].float()).all(), r
            assert hit or torch.isfinite(out[r].float()).all(), r


@pytest.mark.gpu
def test_a_long_context_in_chunks_of_keys(ops):
    """Few rows behind a long context: the keys of the kernel over pages read back are cut, and the parts merged."""
    c = make(ops, BF, 2, 1, 128, 16, [17000], [70], seed=3)
    check(c, prefill(ops, c, work=True), 128 ** -0.5, rows=[0, 1, 33, 68, 69])
    check(c, prefill(ops, c, 16500, work=True), 128 ** -0.5, 16500, rows=[0, 69])


@pytest.mark.gpu
@pytest.mark.parametrize("kw", EXTRAS)
def test_long_chunk_extras(ops, kw):
    kw, told, window, keep = numbers(kw, 4)
    for hd in (64, 96):
        c = make(ops, BF, 4, 2, hd, 16, [190, 300], [120, 90], seed=hd)
        check(c, prefill(ops, c, window, work=True, **kw), hd ** -0.5, window, keep, rows=list(range(0, 210, 11)) + [119, 120, 209], **told)


@pytest.mark.gpu
def test_rows_of_other_requests_stay(ops):
    """A step holds decoding rows first: the chunks' call starts at a later request and row and leaves the others' results."""
    for work in (False, True):
        c = make(ops, BF, 4, 2, 64, 16, [90, 33, 200, 140], [1, 1, 70 if work else 9, 5], seed=3)
        out = prefill(ops, c, work=work, seg0=2)
        assert torch.all(out[:2] == 7.5)
        check(c, out, 1 / 8, rows=list(range(2, len(c["positions"]), 3)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_masked_places_may_hold_anything(ops, dtype):
    """NaN in free slots (every test here), values of one sign, large scores, and a key far back that takes all the weight."""
    c = make(ops, dtype, 2, 2, 64, 16, [500, 31], [1, 1], seed=6, spread=30.0)
    check(c, decode(ops, c), 1 / 8)
    for x in range(2):
        c["held"][x][0] = c["held"][x][0].abs()
    c["k"].codes.abs_()
    c["v"].codes.abs_()
    c["held"][0][1], c["held"][1][1] = c["held"][0][1].abs(), c["held"][1][1].abs()
    check(c, decode(ops, c), 1 / 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_key_that_is_not_finite(ops, dtype):
    """A key or value written from a NaN is NaN to the rows that see it and to no other."""
    for x in "kv":
        c = make(ops, dtype, 4, 2, 64, 16, [100, 100], [20, 20], seed=8)
        c[x].scales[int(c["table"][0, 90 // 16]), 1, 90 % 16] = math.nan
        out = prefill(ops, c).cpu().view(40, 4, 64)
        for r in range(40):
            hit = r < 20 and 80 + r >= 90
            assert torch.isnan(out[r, 2:]).all().item() == hit and torch.isfinite(out[r, :2].float()).all()
            assert hit or torch.isfinite(out[r].float()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ps", [16, 5])
def test_pages_that_the_cache_does_not_have(ops, dtype, ps):
    """A page number outside the cache is passed over; a row all of whose pages are such sees nothing and gets zeros, and so does
    one of a request outside the table, or one behind the table's last block only as far as that goes."""
    c = make(ops, dtype, 2, 2, 32, ps, [100, 60, 40], [1, 1, 1], seed=1)
    c["table"][0, 2], c["table"][0, 0] = -1, 10 ** 6
    c["table"][1] = -7
    gone = set(range(0, ps)) | set(range(2 * ps, 3 * ps))
    out = decode(ops, c)
    assert torch.all(out[1] == 0)
    for r, keys in ((0, [j for j in range(100) if j not in gone]), (2, list(range(40)))):
        for h in range(2):
            ref, weighted, size = plain_q8.attend(c["q"][r, h * 32:h * 32 + 32].double(), c["held"][0][r][:, h], c["held"][1][r][:, h], 99 if r == 0 else 39, keys, 32 ** -0.5)
            assert ((out[r, h * 32:h * 32 + 32].double().cpu() - ref).abs() <= plain_q8.tolerance(dtype, ref, weighted, size, 32, len(keys))).all()
    seq = torch.tensor([5, 2 ** 31 - 1, 2], dtype=torch.int32)
    out = decode(ops, c, seq=seq)
    assert torch.all(out[:2] == 0) and torch.any(out[2] != 0)
    far = dict(c, positions=torch.tensor([2 ** 31 - 1, -5, 39], dtype=torch.int32), seq=torch.tensor([2, 2, 2], dtype=torch.int32))
    out = decode(ops, far, max_context=100)
    # at that position the row sees every slot of the request's pages: the free ones, if the last page has any, hold NaN here
    assert torch.all(out[1] == 0) and torch.isnan(out[0]).all().item() == (40 % ps != 0) and torch.isfinite(out[2].float()).all()


@pytest.mark.gpu
def test_strided_rows_another_stream_and_a_captured_step(ops):
    """Rows inside wider ones; a call on a stream of its own; two captured steps that share their scratch, replayed in turn."""
    c = make(ops, BF, 6, 3, 128, 16, [700, 90, 333], [1, 1, 1], seed=5)
    wide = torch.zeros(3, 6 * 128 + 64, dtype=BF, device="cuda")
    wide[:, :6 * 128] = c["q"].cuda()
    out = torch.full((3, 6 * 128 + 16), 2.5, dtype=BF, device="cuda")
    decode(ops, c, q=wide, out=out)
    check(c, out[:, :6 * 128], 128 ** -0.5)
    assert torch.all(out[:, 6 * 128:] == 2.5)
    buf = scratch(ops, 3, 1, 0, c)
    args = dict(k=c["k"], v=c["v"])
    table, seq, pos, q = c["table"].cuda(), c["seq"].cuda(), c["positions"].cuda(), c["q"].cuda()
    outs = [torch.zeros(3, 6 * 128, dtype=BF, device="cuda") for _ in range(3)]

    def call(o, window):
        ops.paged_decode_q8(q, -1, -1, args["k"], args["v"], table, seq, pos, None, o, *buf, 6, 3, 128, 16, 128 ** -0.5, window, 700)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(outs[0], 0)
    torch.cuda.current_stream().wait_stream(side)
    check(c, outs[0], 128 ** -0.5)
    graphs = []
    for o, window in ((outs[1], 0), (outs[2], 64)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(o, window)
        graphs.append(gr)
    for _ in range(3):
        for gr in graphs:
            gr.replay()
    q.copy_(q.flip(0))      # new queries for the captured steps
    c["q"] = c["q"].flip(0)
    for gr in graphs:
        gr.replay()
    check(c, outs[1], 128 ** -0.5)
    check(c, outs[2], 128 ** -0.5, 64)


@pytest.mark.gpu
def test_the_same_result_every_time(ops):
    """Pieces of a row are joined in one order whoever is last."""
    c = make(ops, BF, 8, 2, 128, 16, [3000, 40, 1777], [1, 1, 1], seed=7)
    first = decode(ops, c)
    for _ in range(20):
        assert torch.equal(decode(ops, c), first)


@pytest.mark.gpu
def test_store_attend_and_read_back_together(ops):
    """As a server uses them: a prompt in two portions, then tokens one by one, all against the values that the cache stands for."""
    g = torch.Generator().manual_seed(11)
    H, G, hd, ps, n = 4, 2, 64, 16, 180
    wide = (H + 2 * G) * hd
    qkv = torch.randn(n, wide, generator=g).to(BF)
    c = dict(H=H, G=G, hd=hd, ps=ps, dtype=BF, k=ops.q8_pages(14, G, ps, hd), v=ops.q8_pages(14, G, ps, hd),
             table=torch.randperm(14, generator=g)[None, :12].to(torch.int32), q=qkv[:, :H * hd], ctx=[n])
    c["held"] = [[], []]
    for x, off in ((0, H * hd), (1, (H + G) * hd)):
        code, scale = plain_q8.quantise(qkv[:, off:off + G * hd].view(n, G, hd))
        c["held"][x].append(code * scale.double()[..., None])
    pos = torch.arange(n, dtype=torch.int32)
    slots = (c["table"][0, (pos // ps).long()] * ps + pos % ps).cuda()
    rows, table = qkv.cuda(), c["table"].cuda()
    out = torch.full((n, H * hd), math.nan, dtype=BF, device="cuda")
    work = tuple(torch.full((14, G, ps, hd), math.nan, dtype=BF, device="cuda") for _ in "kv")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    floats, counters = ops.attention_q8_scratch(150, 150, 1, H, G, hd, n, BF)
    buf = torch.empty(floats, device="cuda"), torch.zeros(counters, dtype=torch.int32, device="cuda")
    for a, b in ((0, 23), (23, 173)):
        ops.kv_write_q8(rows[a:b], H * hd, (H + G) * hd, c["k"], c["v"], slots[a:b], G, hd, ps)
        ops.paged_prefill_q8(rows[a:b], c["k"], c["v"], table, i32(0, b - a), i32(a), i32(b), pos[a:b].cuda(), out[a:b], 0, 1, 0, b - a, b - a, H, G, hd, ps,
                             hd ** -0.5, 0, b, *buf, work)
    dec = scratch(ops, 1, 1, 0, c)
    for p in range(173, n):
        ops.paged_decode_q8(rows[p:p + 1], H * hd, (H + G) * hd, c["k"], c["v"], table, i32(0), i32(p), slots[p:p + 1], out[p:p + 1], *dec, H, G, hd, ps,
                            hd ** -0.5, 0, n)
    c.update(seq=torch.zeros(n, dtype=torch.int32), positions=pos)
    check(c, out, hd ** -0.5, rows=list(range(23)) + list(range(23, 173, 7)) + list(range(173, n)))
    ko, vo = (torch.zeros(14, G, ps, hd, device="cuda") for _ in "kv")
    ops.kv_read_q8(c["k"], c["v"], ko, vo, table, i32(0), i32(n), n)
    assert torch.equal(ko[table[0].long()].transpose(1, 2).reshape(-1, G, hd)[:n].double().cpu(), c["held"][0][0].float().double())


def test_refusals():
    from cbis_b200.kernels import ops
    H, G, hd, ps = 4, 2, 32, 16
    kp, vp = ops.q8_pages(2, G, ps, hd, device="cpu"), ops.q8_pages(2, G, ps, hd, device="cpu")
    q, out = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 128, dtype=BF)
    i, table = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32)
    f = torch.zeros(1 << 16)
    good = dict(qkv=q, k_off=128, v_off=192, k_pages=kp, v_pages=vp, block_table=table, row_seq=i, positions=i, slot_mapping=i, out=out, scratch=f,
                counters=i, n_head=H, n_kv_head=G, head_dim=hd, page_size=ps, scale=1.0, window=0, max_context=32)
    bad = [("no CPU path", {}), ("is not supported", dict(qkv=q.half())), ("multiple of 16", dict(head_dim=24)), ("multiple of 16", dict(head_dim=272)),
           ("not a multiple of n_kv_head", dict(n_head=3)), ("keys' codes", dict(page_size=8)), ("int8 codes", dict(v_pages=ops.Q8Pages(vp.codes.int(), vp.scales))),
           ("different numbers", dict(v_pages=ops.q8_pages(3, G, ps, hd, device="cpu"))), ("block table", dict(block_table=table.long())),
           ("do not fit rows", dict(qkv=q[:, :100])), ("out must", dict(out=out.float())), ("out must", dict(out=out[:2])), ("scratch", dict(scratch=f.double())),
           ("counters", dict(counters=i.long())), ("sinks must", dict(sinks=torch.zeros(3))), ("rates need", dict(rates=torch.zeros(4))),
           ("keep", dict(keep=-1)), ("row_seq", dict(row_seq=i[:2])), ("positions", dict(positions=i.float())), ("do not lie in rows", dict(v_off=200)),
           ("slot_mapping", dict(slot_mapping=None))]
    for match, change in bad:
        with pytest.raises(ops.KernelError, match=match):
            ops.paged_decode_q8(**{**good, **change})
    good = dict(q=q, k_pages=kp, v_pages=vp, block_table=table, cu_rows=i, seg_start=i, seg_ctx=i, positions=i, out=out, seg0=0, n_seg=2, row0=0, n_rows=3,
                max_seg_rows=2, n_head=H, n_kv_head=G, head_dim=hd, page_size=ps, scale=1.0, window=0, max_context=32, scratch=f, counters=i)
    bad = [("no CPU path", {}), ("not in the block table", dict(n_seg=3)), ("not in the block table", dict(seg0=-1)), ("are not in q", dict(n_rows=4)),
           ("cu_rows", dict(cu_rows=i[:2])), ("seg_start", dict(seg_start=i[:1])), ("seg_ctx", dict(seg_ctx=i[:1])), ("positions", dict(positions=i[:2])),
           ("work must", dict(work=(torch.zeros(2, G, ps, hd), torch.zeros(2, G, ps, hd)))), ("multiple of 16", dict(head_dim=40))]
    for match, change in bad:
        with pytest.raises(ops.KernelError, match=match):
            ops.paged_prefill_q8(**{**good, **change})


@pytest.mark.gpu
def test_refusals_of_the_launcher(ops):
    c = make(ops, BF, 2, 2, 32, 16, [40], [1], seed=1)
    floats, counters = ops.attention_q8_scratch(1, 1, 0, 2, 2, 32, 40, BF)
    for buf in ((floats - 1, counters), (floats, counters - 1)):
        with pytest.raises(ops.KernelError, match="a size"):
            decode(ops, c, buffers=(torch.zeros(buf[0], device="cuda"), torch.zeros(buf[1], dtype=torch.int32, device="cuda")))
    with pytest.raises(ops.KernelError, match="misaligned"):
        decode(ops, c, q=torch.zeros(1, 65, dtype=BF, device="cuda")[:, 1:])
    with pytest.raises(ops.KernelError, match="too large"):
        big = torch.zeros(5000, 64, dtype=BF, device="cuda")
        decode(ops, dict(c, positions=torch.zeros(5000, dtype=torch.int32)), q=big, seq=torch.zeros(5000, dtype=torch.int32),
               buffers=(torch.zeros(1 << 22, device="cuda"), torch.zeros(1 << 15, dtype=torch.int32, device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_numbers_behind_every_position(ops, dtype):
    """A window, kept keys and a context that no position reaches, beyond 32 bits too, are those of a call without a limit."""
    c = make(ops, dtype, 2, 2, 32, 16, [90, 33], [1, 1], seed=2)
    plain = decode(ops, c)
    for far in (2 ** 30, 2 ** 31 + 5, 2 ** 32 + 40):
        assert torch.equal(decode(ops, c, far), plain)
        assert torch.equal(decode(ops, c, 0, max_context=90, buffers=scratch(ops, 2, 1, 0, c), keep=far), plain)
        # (kept first keys are seen by every row: the window's start is then no limit)
        check(c, decode(ops, c, 20, keep=far), 32 ** -0.5, 20, 90)
    with pytest.raises(ops.KernelError, match="a size"):
        decode(ops, c, -2 ** 31)
    c = make(ops, dtype, 2, 2, 64, 16, [190, 130], [150, 90], seed=2)
    for far in (2 ** 30, 2 ** 31 + 5, 2 ** 32 + 40):
        check(c, prefill(ops, c, far), 1 / 8, rows=[0, 149, 150, 239])
        if dtype == BF:
            check(c, prefill(ops, c, far, work=True, keep=far), 1 / 8, rows=[0, 149, 150, 239])


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_a_page_that_the_cache_does_not_have_in_a_long_chunk(ops, hd):
    """Over pages read back such a page holds nothing: the rows that see it get not-a-numbers, the others their results."""
    for page in (-1, 10 ** 6):
        c = make(ops, BF, 4, 2, hd, 16, [300, 260], [150, 140], seed=9)
        c["table"][0, 200 // 16] = page
        out = prefill(ops, c, work=True)
        for r in range(290):
            hit = r < 150 and 150 + r >= 192
            assert torch.isnan(out[r].float()).all().item() == hit, r
        check(c, out, hd ** -0.5, rows=[0, 41, 150, 200, 289])


@pytest.mark.gpu
def test_two_calls_at_once(ops):
    """On two streams, each with scratch and counters of its own."""
    cs = [make(ops, BF, 8, 2, 128, 16, [3000, 40, 1777], [1, 1, 1], seed=s) for s in (7, 8)]
    alone = [decode(ops, c) for c in cs]
    fixed = [(c["q"].cuda(), c["table"].cuda(), c["seq"].cuda(), c["positions"].cuda(), torch.zeros_like(alone[0]), scratch(ops, 3, 1, 0, c)) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(10):
        for c, (q, table, seq, pos, out, buf), stream in zip(cs, fixed, streams):
            with torch.cuda.stream(stream):
                ops.paged_decode_q8(q, -1, -1, c["k"], c["v"], table, seq, pos, None, out, *buf, 8, 2, 128, 16, 128 ** -0.5, 0, 3000)
    torch.cuda.synchronize()
    for (_, _, _, _, out, _), ref in zip(fixed, alone):
        assert torch.equal(out, ref)


@pytest.mark.gpu
def test_scratch_of_a_long_chunk(ops):
    """The parts of a long context need room: less is refused before anything is launched."""
    c = make(ops, BF, 2, 1, 128, 16, [9000], [70], seed=3)
    work = tuple(torch.zeros(c["k"].codes.shape, dtype=BF, device="cuda") for _ in "kv")
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    out = torch.full(c["q"].shape, 7.5, dtype=BF, device="cuda")
    floats, counters = ops.attention_q8_scratch(70, 70, 1, 2, 1, 128, 9000, BF)
    takes, ops.prefill_q8_reads_back = ops.prefill_q8_reads_back, lambda *a: True
    try:
        with pytest.raises(ops.KernelError, match="scratch has"):
            ops.paged_prefill_q8(c["q"].cuda(), c["k"], c["v"], c["table"].cuda(), c["cu"].cuda(), i32(8930), i32(9000), c["positions"].cuda(), out, 0, 1, 0,
                                 70, 70, 2, 1, 128, 16, 1.0, 0, 9000, torch.zeros(100, device="cuda"), torch.zeros(counters, dtype=torch.int32, device="cuda"), work)
    finally:
        ops.prefill_q8_reads_back = takes
    assert torch.all(out == 7.5) and not any(w.any() for w in work)


def test_one_array_is_not_stored_twice():
    """Both of a token's rows would go to one place."""
    from cbis_b200.kernels import ops
    p = ops.q8_pages(2, 2, 16, 32, device="cpu")
    q, out = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 128, dtype=BF)
    i, table, f = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(1 << 16)
    for v in (p, ops.Q8Pages(p.codes.view(p.codes.shape), p.scales)):
        with pytest.raises(ops.KernelError, match="of one array"):
            ops.paged_decode_q8(q, 128, 192, p, v, table, i, i, i, out, f, i, 4, 2, 32, 16, 1.0, 0, 32)


def test_values_that_are_not_given_are_refused():
    """Writing and reading back take None for one array of both; attention wants the values' pages named."""
    from cbis_b200.kernels import ops
    p = ops.q8_pages(2, 2, 16, 32, device="cpu")
    q, out = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 128, dtype=BF)
    i, table, f = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(1 << 16)
    with pytest.raises(ops.KernelError, match="without values' pages"):
        ops.paged_decode_q8(q, -1, -1, p, None, table, i, i, i, out, f, i, 4, 2, 32, 16, 1.0, 0, 32)
    with pytest.raises(ops.KernelError, match="without values' pages"):
        ops.paged_prefill_q8(q, p, None, table, i, i, i, i, out, 0, 2, 0, 3, 2, 4, 2, 32, 16, 1.0, 0, 32, f, i)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n", [1, 17, 33, 700])
def test_the_only_key_of_a_tile_is_not_finite(ops, dtype, n):
    """The newest key is the first of its tile, or the only one that the row sees: what a warp or block has of it is not-a-number with no
    maximum, and the join has to keep that."""
    for x in "kv":
        c = make(ops, dtype, 4, 2, 64, 16, [n, 20], [1, 1], seed=n)
        c[x].scales[int(c["table"][0, (n - 1) // 16]), 1, (n - 1) % 16] = math.nan
        out = decode(ops, c).cpu().float().view(2, 4, 64)
        assert torch.isnan(out[0, 2:]).all() and torch.isfinite(out[0, :2]).all() and torch.isfinite(out[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("hd", [64, 128])
def test_the_first_key_of_a_long_chunk_is_not_finite(ops, hd):
    """Row 0 sees this key alone, and behind a window of 50 later rows do not see it."""
    for x in "kv":
        c = make(ops, BF, 4, 2, hd, 16, [200], [200], seed=hd)
        c[x].scales[int(c["table"][0, 0]), 1, 0] = math.nan
        for window, seen in ((0, 200), (50, 50)):
            out = prefill(ops, c, window, work=True).cpu().float().view(200, 4, hd)
            assert torch.isfinite(out[:, :2]).all() and torch.isnan(out[:seen, 2:]).all() and torch.isfinite(out[seen:]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,hd", [(8, 256), (16, 256), (16, 144), (8, 128), (4, 32)])
def test_as_many_rows_as_a_call_takes(ops, dtype, H, hd):
    """The rows' list lies in shared memory beside the tiles: with ``ATTENTION_Q8_MAX_ROWS`` of them the block is at its largest."""
    n = ops.ATTENTION_Q8_MAX_ROWS
    g = torch.Generator().manual_seed(hd)
    c = make(ops, dtype, H, 1, hd, 16, [33, 1, 90, 200], [1] * 4, seed=H)
    seq = torch.randint(0, 4, (n,), generator=g)
    positions = (torch.rand(n, generator=g) * torch.tensor(c["ctx"])[seq]).to(torch.int32)
    c.update(q=torch.randn(n, H * hd, generator=g).to(dtype), seq=seq.to(torch.int32), positions=positions)
    check(c, decode(ops, c), hd ** -0.5, rows=[0, 1, n // 2, n - 2, n - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
def test_as_many_row_tiles_as_a_call_takes(ops, dtype):
    """A chunk of one row a tile (16 query heads over one; in 32 bits at this width 8)."""
    n, H = ops.ATTENTION_Q8_MAX_ROWS, 16 if dtype == BF else 8
    c = make(ops, dtype, H, 1, 256, 64, [n], [n], seed=3)
    assert ops.prefill_q8_takes(n, n, 1, H, 1, 256, 64, dtype)
    check(c, prefill(ops, c), 1 / 16, rows=[0, 1, 2000, n - 1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps", [(4, 2, 64, 16), (3, 3, 32, 5), (12, 1, 128, 16)])
def test_a_head_without_a_sink(ops, dtype, H, G, hd, ps):
    """Its number is -inf: rows that see something get what they get without a sink, the others zeros, whether one block has the row's keys or
    many (the third row's pages are all absent, the fourth row is of no request)."""
    c = make(ops, dtype, H, G, hd, ps, [40, 3000, 3000, 1, 20], [1] * 5, seed=H)
    c["table"][2], c["table"][4] = -1, -1
    c["seq"][3] = -1
    sinks = torch.tensor([-math.inf if h != 1 else 0.3 for h in range(H)])
    out = decode(ops, c, sinks=sinks.cuda())
    assert torch.all(out[2:] == 0)
    check(c, out, hd ** -0.5, rows=[0, 1], sink=sinks.tolist())
    c = make(ops, dtype, H, G, hd, ps, [90, 60], [7, 9], seed=H)
    c["table"][1] = -1
    out = prefill(ops, c, sinks=sinks.cuda())
    assert torch.all(out[7:] == 0)
    check(c, out, hd ** -0.5, rows=range(7), sink=sinks.tolist())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("H,G,hd,ps", [(4, 2, 64, 16), (3, 3, 48, 5)])
def test_kept_keys_of_a_row_behind_the_table(ops, dtype, H, G, hd, ps):
    """A position behind the block table's last block sees what it would if the table went on with pages that are not there: of the
    window what lies in the table, and the kept first keys."""
    c = make(ops, dtype, H, G, hd, ps, [160, 160, 160, 160], [1] * 4, seed=hd)
    c["table"] = c["table"][:, :-(-160 // ps)].contiguous()
    end, window, keep = 160, 40, 19
    c["positions"] = torch.tensor([159, end + 20, end + 1000, 2 ** 31 - 1], dtype=torch.int32)
    seen = [[*range(keep), *range(120, 160)], [*range(keep), *range(end + 20 - 39, end)], [*range(keep)], [*range(keep)]]
    out = decode(ops, c, window, max_context=160, keep=keep).double().cpu()
    start = c["positions"].clamp_max(2 ** 30).cuda()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    rows = torch.full_like(c["q"].cuda(), math.nan)
    ops.paged_prefill_q8(c["q"].cuda(), c["k"], c["v"], c["table"].cuda(), i32(0, 1, 2, 3, 4), start, start + 1, start, rows, 0, 4, 0, 4, 1, H, G, hd, ps, hd ** -0.5,
                         window, 160, *scratch(ops, 4, 1, 4, c), keep=keep)
    for r, keys in enumerate(seen):
        for h in range(H):
            cols = slice(h * hd, (h + 1) * hd)
            ref, weighted, size = plain_q8.attend(c["q"][r, cols].double(), c["held"][0][r][:, h // (H // G)], c["held"][1][r][:, h // (H // G)], 159, keys, hd ** -0.5)
            tol = plain_q8.tolerance(dtype, ref, weighted, size, hd, len(keys))
            assert ((out[r, cols] - ref).abs() <= tol).all() and ((rows[r, cols].double().cpu() - ref).abs() <= tol).all(), (r, h)


def test_keys_and_values_are_not_read_back_into_the_same_pages():
    from cbis_b200.kernels import ops
    kp, vp = ops.q8_pages(2, 2, 16, 32, device="cpu"), ops.q8_pages(2, 2, 16, 32, device="cpu")
    q, out, w = torch.zeros(3, 256, dtype=BF), torch.zeros(3, 128, dtype=BF), torch.zeros(2, 2, 16, 32, dtype=BF)
    i, table, f = torch.zeros(4, dtype=torch.int32), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(1 << 16)
    with pytest.raises(ops.KernelError, match="the same pages"):
        ops.kv_read_q8(kp, vp, w, w, table, i, i, 32)
    call = lambda v, work: ops.paged_prefill_q8(q, kp, v, table, i, i, i, i, out, 0, 2, 0, 3, 2, 4, 2, 32, 16, 1.0, 0, 32, f, i, work)      # noqa: E731
    with pytest.raises(ops.KernelError, match="the same pages"):
        call(vp, (w, w))
    for v, work in ((kp, (w, w)), (vp, (w, w.clone()))):      # one array for both may go to one place
        with pytest.raises(ops.KernelError, match="no CPU path"):
            call(v, work)
