"""The 8-bit cache: rows written as codes and scales, and read back."""
import math

import pytest
import torch

import plain_q8

TYPES = [torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    from cbis_b200.kernels import ops as o
    return o


def rows_that_are_hard(n, width, dtype, g):
    """Rows of ordinary numbers, and rows where quantising goes wrong most easily."""
    x = torch.randn(n, width, generator=g)
    x[0] = 0.0
    x[1] *= 1e-36                                     # below the scale's floor
    x[2] *= 1e30
    x[3] = torch.round(x[3] * 4) / 4                  # many equal numbers
    if width >= 8:
        x[4, :8] = torch.tensor([2.0, 1.0, -1.0, -2.0, 0.5, 0.0, -0.0, 1.5])      # half of the largest lies on a half step
        x[5, :4] = torch.tensor([254.0, 1.0, -3.0, 127.0])                        # scale 2: half steps of whole numbers
        x[5, 4:] = torch.arange(width - 4) % 254 - 120
    x[6, width // 2] = math.inf
    x[7, width - 1] = math.nan
    x[8] = 2.0 ** -133                                # subnormal in both types
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("heads,hd,vd,ps", [(1, 8, 8, 1), (3, 24, 24, 8), (8, 32, 32, 16), (25, 64, 64, 16), (2, 80, 48, 4), (2, 128, 128, 16),
                                            (3, 7, 13, 5), (1, 256, 128, 32), (1, 576, 64, 16), (2, 200, 200, 3)])
def test_write_and_read(ops, dtype, heads, hd, vd, ps):
    g = torch.Generator().manual_seed(hd * 7 + ps)
    T, pages = 23, 9
    k, v = (rows_that_are_hard(T * heads, w, dtype, g).view(T, heads, w) for w in (hd, vd))
    order = torch.randperm(pages * ps, generator=g)
    slots = torch.full((T,), -1, dtype=torch.int32)
    n = min(T, pages * ps)
    slots[:n] = order[:n].to(torch.int32)
    slots[T - 1], slots[T - 2], slots[T - 3] = -1, pages * ps, 2 ** 31 - 1      # none of these is a slot of the cache
    off_k = 16
    off_v = -(-(off_k + heads * hd) // 8) * 8 + 8
    wide = -(-(off_v + heads * vd) // 8) * 8 + 8
    qkv = torch.full((T, wide), 7.0, dtype=dtype)
    qkv[:, off_k:off_k + heads * hd] = k.reshape(T, -1)
    qkv[:, off_v:off_v + heads * vd] = v.reshape(T, -1)
    kp, vp = ops.q8_pages(pages, heads, ps, hd), ops.q8_pages(pages, heads, ps, vd)
    for p in (kp, vp):
        p.codes.fill_(99)
        p.scales.fill_(0.5)
    ops.kv_write_q8(qkv.cuda(), off_k, off_v, kp, vp, slots.cuda(), heads, hd, ps, vd)
    for x, p, w in ((k, kp, hd), (v, vp, vd)):
        codes = torch.full((pages, heads, ps, w), 99.0, dtype=torch.float64)
        scales = torch.full((pages, heads, ps), 0.5)
        c, s = plain_q8.quantise(x)
        for t in range(T):
            if 0 <= slots[t] < pages * ps:
                codes[int(slots[t]) // ps, :, int(slots[t]) % ps] = c[t]
                scales[int(slots[t]) // ps, :, int(slots[t]) % ps] = s[t]
        assert torch.equal(p.codes.cpu().double(), codes)
        assert torch.equal(torch.nan_to_num(p.scales.cpu(), nan=-1.0), torch.nan_to_num(scales, nan=-1.0))
    # read back: two requests over some of the pages, one of them with a page given back and a page number that is none
    mb = 4
    table = torch.tensor([[3, 1, -1, 5], [0, 99, 2, -1]], dtype=torch.int32)
    start, ctx = torch.tensor([2 * ps, ps // 2], dtype=torch.int32), torch.tensor([4 * ps - ps // 3, 3 * ps], dtype=torch.int32)
    for window, keep, whole in ((0, 0, False), (ps + 1, 0, False), (1, 0, False), (ps + 1, 2, True), (-2 * ps, 1, False)):
        ko, vo = (torch.full((pages, heads, ps, w), 3.25, dtype=dtype, device="cuda") for w in (hd, vd))
        ops.kv_read_q8(kp, vp, ko, vo, table.cuda(), start.cuda(), ctx.cuda(), mb * ps, window, keep, whole_pages=whole)
        for p, o, w in ((kp, ko, hd), (vp, vo, vd)):
            values = (p.codes.cpu().float() * p.scales.cpu()[..., None]).to(dtype)
            want = torch.full((pages, heads, ps, w), 3.25, dtype=dtype)
            for r in range(2):
                seen = {j for q in range(int(start[r]), int(ctx[r])) for j in plain_q8.seen_keys(q, window, keep)}
                if whole:
                    seen = {j for j in range(int(ctx[r])) if any(i // ps == j // ps for i in seen)}
                for j in seen:
                    page = int(table[r, j // ps])
                    if 0 <= page < pages:
                        want[page, :, j % ps] = values[page, :, j % ps]
            assert torch.equal(torch.nan_to_num(o.cpu().float(), nan=-9.0), torch.nan_to_num(want.float(), nan=-9.0)), (window, keep, whole)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_every_row_of_its_values(ops, dtype):
    """Many rows at once: the codes are the nearest ones by the exact quotient, none is off by a step."""
    g = torch.Generator(device="cuda").manual_seed(5)
    T, heads, hd, ps = 4096, 4, 64, 16
    x = torch.randn(T, 2 * heads * hd, device="cuda", generator=g).mul_(torch.exp(2 * torch.randn(T, 1, device="cuda", generator=g))).to(dtype)
    kp, vp = ops.q8_pages(T // ps, heads, ps, hd), ops.q8_pages(T // ps, heads, ps, hd)
    ops.kv_write_q8(x, 0, heads * hd, kp, vp, torch.arange(T, dtype=torch.int32, device="cuda"), heads, hd, ps)
    for p, part in ((kp, x[:, :heads * hd]), (vp, x[:, heads * hd:])):
        c, s = plain_q8.quantise(part.reshape(T, heads, hd))
        assert torch.equal(p.scales.permute(0, 2, 1).reshape(T, heads), s)
        assert torch.equal(p.codes.permute(0, 2, 1, 3).reshape(T, heads, hd).double(), c)


@pytest.mark.gpu
def test_one_array_for_keys_and_values(ops):
    g = torch.Generator().manual_seed(3)
    kp = ops.q8_pages(3, 1, 16, 72)
    x = torch.randn(20, 80, generator=g).to(torch.bfloat16)
    slots = torch.randperm(48, generator=g)[:20].to(torch.int32)
    for values in (None, kp):
        kp.codes.zero_()
        ops.kv_write_q8(x.cuda(), 8, 8, kp, values, slots.cuda(), 1, 72, 16, 64)
        c, s = plain_q8.quantise(x[:, 8:])
        flat = kp.codes.cpu().view(48, 72)[slots.long()]
        assert torch.equal(flat.double(), c) and torch.equal(kp.scales.cpu().view(48)[slots.long()], s)
    out = torch.zeros(3, 1, 16, 72, dtype=torch.bfloat16, device="cuda")
    table, start = torch.tensor([[0, 1, 2]], dtype=torch.int32).cuda(), torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_read_q8(kp, kp, out, None, table, start, start + 48, 48)
    assert torch.equal(out.cpu(), (kp.codes.cpu().float() * kp.scales.cpu()[..., None]).to(torch.bfloat16))


@pytest.mark.gpu
def test_empty_calls(ops):
    kp, vp = ops.q8_pages(2, 1, 16, 16), ops.q8_pages(2, 1, 16, 16)
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv_write_q8(torch.zeros(0, 32, dtype=torch.bfloat16, device="cuda"), 0, 16, kp, vp, i[:0], 1, 16, 16)
    ko, vo = (torch.full((2, 1, 16, 16), 1.5, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    ops.kv_read_q8(kp, vp, ko, vo, table, i, i, 32)                 # a request without tokens
    ops.kv_read_q8(kp, vp, ko, vo, table[:0], i[:0], i[:0], 32)     # no request
    assert torch.all(ko == 1.5) and torch.all(vo == 1.5)


def test_refusals():
    from cbis_b200.kernels import ops
    kp, vp = ops.q8_pages(2, 2, 16, 32, device="cpu"), ops.q8_pages(2, 2, 16, 32, device="cpu")
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    slots = torch.zeros(3, dtype=torch.int32)

    def refused(match, *a, **k):
        with pytest.raises(ops.KernelError, match=match):
            ops.kv_write_q8(*a, **k)

    refused("no CPU path", x, 0, 64, kp, vp, slots, 2, 32, 16)
    refused("is not supported", x.half(), 0, 64, kp, vp, slots, 2, 32, 16)
    refused("do not lie in rows", x, 0, 96, kp, vp, slots, 2, 32, 16)
    refused("do not lie in rows", x, -1, 64, kp, vp, slots, 2, 32, 16)
    refused("do not lie in rows", x.t().contiguous().t(), 0, 64, kp, vp, slots, 2, 32, 16)
    refused("keys' codes", x, 0, 64, kp, vp, slots, 2, 32, 8)
    refused("values' codes", x, 0, 64, kp, ops.Q8Pages(vp.codes[..., :16], vp.scales), slots, 2, 32, 16)
    refused("int8 codes", x, 0, 64, ops.Q8Pages(kp.codes.float(), kp.scales), vp, slots, 2, 32, 16)
    refused("scales are not", x, 0, 64, ops.Q8Pages(kp.codes, kp.scales[:1]), vp, slots, 2, 32, 16)
    refused("different numbers", x, 0, 64, kp, ops.q8_pages(3, 2, 16, 32, device="cpu"), slots, 2, 32, 16)
    refused("slot_mapping", x, 0, 64, kp, vp, slots[:2], 2, 32, 16)
    refused("slot_mapping", x, 0, 64, kp, vp, slots.long(), 2, 32, 16)

    ko, vo = torch.zeros(2, 2, 16, 32), torch.zeros(2, 2, 16, 32)
    table, i = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)

    def unread(match, *a, **k):
        with pytest.raises(ops.KernelError, match=match):
            ops.kv_read_q8(*a, **k)

    unread("no CPU path", kp, vp, ko, vo, table, i, i, 32)
    unread("is not supported", kp, vp, ko.half(), vo.half(), table, i, i, 32)
    unread("of one type", kp, vp, ko, vo.bfloat16(), table, i, i, 32)
    unread("of one type", kp, vp, ko, vo[:1], table, i, i, 32)
    unread("block table", kp, vp, ko, vo, table[0], i, i, 32)
    unread("seg_ctx", kp, vp, ko, vo, table, i, i[:0], 32)
    unread("keep", kp, vp, ko, vo, table, i, i, 32, 8, -1)


def test_the_plain_form_rounds_half_steps_to_even():
    c, s = plain_q8.quantise(torch.tensor([[254.0, 1.0, 3.0, -1.0, -5.0, 127.0]]))
    assert s.item() == 2.0 and c.tolist() == [[127.0, 0.0, 2.0, 0.0, -2.0, 64.0]]


@pytest.mark.gpu
def test_pages_read_back_are_there_for_the_kernel_behind(ops):
    """The decode kernel asks for its first keys before it waits for the kernel ahead: read back and attended to one right after the other,
    over pages that hold other numbers each time, the results are those of a stop in between."""
    g = torch.Generator().manual_seed(2)
    H, hd, ps, S, blocks = 8, 128, 16, 4, 24
    pages = S * blocks
    kp, vp = ops.q8_pages(pages, H, ps, hd), ops.q8_pages(pages, H, ps, hd)
    ko, vo = (torch.zeros(pages, H, ps, hd, dtype=torch.bfloat16, device="cuda") for _ in "kv")
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")      # noqa: E731
    table = torch.randperm(pages, generator=g).view(S, blocks).to(torch.int32).cuda()
    ctx, seq, none = i32([384, 37, 200, 1]), i32([0, 1, 2, 3]), i32([-1] * 4)
    q = torch.randn(S, H * hd, generator=g).to(torch.bfloat16).cuda()
    for turn in range(20):
        for p in (kp, vp):
            p.codes.random_(-127, 128)
            p.scales.uniform_(0.01, 0.03)
        outs = []
        for stop in (False, True):
            out = torch.empty(S, H * hd, dtype=torch.bfloat16, device="cuda")
            ko.fill_(turn)
            vo.fill_(turn)
            torch.cuda.synchronize()
            ops.kv_read_q8(kp, vp, ko, vo, table, ctx - 1, ctx, 384, whole_pages=True)
            if stop:
                torch.cuda.synchronize()
            ops.paged_decode_bf16(q, -1, -1, ko, vo, table, seq, ctx - 1, none, out, None, None, H, H, hd, ps, hd ** -0.5, 0, 1)
            outs.append(out)
        assert torch.equal(*outs)
