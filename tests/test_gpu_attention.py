"""qkv_norm_rope_append, attn_decode_paged and attn_window against plain 64-bit forms (attention_ref.py derives the
bounds), at the sizes, masks, layouts and contents where they can go wrong."""
import math
import random

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import attention_ref as R  # noqa: E402

BF16, E4M3 = "bf16", "e4m3"


@pytest.fixture(scope="module")
def mx():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    import miroxen_b200 as m
    m.lib()
    m.device_error()
    return m


@pytest.fixture(autouse=True)
def _no_device_error(mx):
    yield
    torch.cuda.synchronize()
    assert mx.device_error() == 0


def rand(g, *shape, std=1.0):
    return (torch.randn(*shape, device="cuda", generator=g) * std).bfloat16()


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_cache(mx, g, kind, seqs, longest, page, Hkv, D, heads_first=False, fill=True, spare=3, scales=True):
    per = max(1, -(-longest // page))
    pages = seqs * per + spare
    shape = (pages, Hkv, page, D) if heads_first else (pages, page, Hkv, D)
    parts, sc = [], []
    for std in (1.2, 1.0):
        if kind == BF16:
            t = rand(g, *shape, std=std) if fill else torch.zeros(shape, device="cuda", dtype=torch.bfloat16)
            sc.append(None)
        else:
            t = (torch.randn(shape, device="cuda", generator=g) * (std * 50 if scales else std)).clamp(-448, 448).to(torch.float8_e4m3fn) if fill else \
                torch.zeros(shape, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
            sc.append(0.01 + 0.02 * torch.rand(Hkv, device="cuda", generator=g) if scales else None)
        parts.append(t.transpose(1, 2) if heads_first else t)
    table = torch.randperm(pages, device="cuda", generator=g)[:seqs * per].view(seqs, per).to(torch.int32)
    return mx.KvCache(parts[0], parts[1], table, sc[0], sc[1])


def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t.view(torch.int16)


# ---- append ---------------------------------------------------------------------------------------------------

def check_append(mx, seed, kind, T, H, Hkv, D, page, rot, mode, packed=False, k_out=True, norm=True, idle=0, seqs=None, heads_first=False,
                 rope_rows=False, odd_table=False):
    g = gen(seed)
    total = T + idle
    seqs = seqs or total
    step = seqs >= total
    room = 3 * page + 1 if step else T + 7
    cache = make_cache(mx, g, kind, seqs, room, page, Hkv, D, heads_first, fill=True)
    before = cache.k.clone(), cache.v.clone()
    if packed:
        buf = rand(g, total, (H + 2 * Hkv) * D)
        q, k, v = buf[:, :H * D], buf[:, H * D:(H + Hkv) * D], buf[:, (H + Hkv) * D:]
    else:
        q, k, v = rand(g, total, H * D), rand(g, total, Hkv * D), rand(g, total, Hkv * D)
    if step:
        ids = torch.randperm(seqs, device="cuda", generator=g)[:total].int()
        pos = torch.randint(0, room, (total,), device="cuda", generator=g).int()
    else:
        ids = (torch.arange(total, device="cuda") % seqs).int()
        pos = (torch.arange(total, device="cuda") // seqs + 5).int()
    if idle:
        ids[torch.randperm(total, device="cuda", generator=g)[:idle]] = -1
    rows = torch.randint(0, 50, (total,), device="cuda", generator=g).int() if rope_rows else None
    table_rows, half = (50 if rope_rows else room), rot // 2
    angle = torch.rand(table_rows, half, device="cuda", generator=g) * 6.3
    cos, sin = angle.cos(), angle.sin()
    if odd_table:  # rows that start off a 16-byte boundary
        cos, sin = (torch.cat([torch.zeros(1, device="cuda"), t.flatten()])[1:].view(table_rows, half) for t in (cos, sin))
    wq, wk = (1 + 0.1 * torch.randn(D, device="cuda", generator=g) if norm else None for _ in range(2))
    q_out = torch.full((total, H, D), 7.0, device="cuda", dtype=torch.bfloat16)
    ko = torch.full((total, Hkv, D), 7.0, device="cuda", dtype=torch.bfloat16) if k_out else None
    mx.qkv_norm_rope_append(q, k, v, total, H, D, wq, wk, 1e-6, cos, sin, table_rows, rot, mode, cache, pos, q_out, seq_ids=ids, rope_rows=rows,
                            k_out=ko, q_stride=q.stride(0), k_stride=k.stride(0), v_stride=v.stride(0))
    live = (ids >= 0).nonzero()[:, 0]
    at = (rows if rope_rows else pos).long()
    # fp32 on the way: the mean of D squares (D 2^-24), a dozen roundings; then one rounding of the result
    rel = (D + 16) * 2.0 ** -24

    def close(got, want, part, what):
        bound = 2.0 ** -8 * want.abs() + (1 + 2.0 ** -8) * rel * part
        R.assert_within(got, want, bound + 1e-30, what)

    wants = {}
    for name, x, w, heads in (("q", q, wq, H), ("k", k, wk, Hkv)):
        x = x.reshape(total, heads, D)
        want = R.rope_reference(x, w, cos[at], sin[at], rot, mode, 1e-6)
        part = want.abs().amax(-1, keepdim=True).expand_as(want) * 2  # of a sum of two products
        wants[name] = want, part
    close(q_out[live], wants["q"][0][live], wants["q"][1][live], "q_out")
    if k_out:
        close(ko[live], wants["k"][0][live], wants["k"][1][live], "k_out")
        assert bool((ko[ids < 0] == 7).all())
    assert bool((q_out[ids < 0] == 7).all())
    page_i = cache.page_table[ids[live].long(), (pos[live] // page).long()].long()
    slot = (pos[live] % page).long()
    for name, t, old, want, scale in (("k", cache.k, before[0], wants["k"], cache.k_scale),
                                      ("v", cache.v, before[1], (v.reshape(total, Hkv, D).double(), None), cache.v_scale)):
        got = raw(t)[page_i, slot].view(t.dtype).double()
        if kind == BF16:
            if name == "v":
                assert torch.equal(got, want[0][live])
            else:
                close(got, want[0][live], want[1][live], "k pages")
        else:
            s = scale.double()[:, None]
            x = (want[0][live] / s).clamp(-448, 448)
            part = torch.zeros_like(x) if want[1] is None else want[1][live] / s
            # half a step: 2^-4 of the value, 2^-10 below the smallest normal 2^-6
            bound = torch.maximum(2.0 ** -4 * x.abs(), torch.full_like(x, 2.0 ** -10)) + 1.07 * ((rel * part) + 2.0 ** -22 * x.abs())
            R.assert_within(got, x, bound, name + " pages")
        # nothing else is touched
        other = raw(t).clone()
        other[page_i, slot] = raw(old)[page_i, slot]
        assert torch.equal(other, raw(old)), name + ": pages outside of the call's rows changed"


APPEND = [
    # kind, T, H, Hkv, D, page, rot, mode
    (BF16, 1, 32, 8, 128, 16, 128, 2), (E4M3, 1, 4, 1, 64, 16, 64, 1), (BF16, 7, 24, 24, 128, 64, 128, 1), (E4M3, 33, 5, 5, 96, 7, 96, 2),
    (BF16, 19, 6, 2, 72, 1, 72, 2), (BF16, 5, 3, 1, 8, 16, 8, 1), (E4M3, 9, 2, 2, 16, 5, 8, 2), (BF16, 13, 7, 7, 80, 24, 40, 2),
    (E4M3, 13, 7, 7, 80, 24, 40, 2), (BF16, 21, 8, 4, 128, 100, 96, 2), (BF16, 4, 8, 4, 128, 100, 6, 1), (BF16, 4, 8, 4, 120, 16, 2, 2),
    (BF16, 3, 70, 70, 128, 16, 128, 2), (E4M3, 3, 1, 1, 128, 256, 0, 2), (BF16, 6, 2, 1, 64, 32, 64, 0)]


@pytest.mark.parametrize("case", APPEND, ids=str)
def test_append(mx, case):
    check_append(mx, 1, *case)


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("more", [dict(packed=True), dict(k_out=False), dict(norm=False), dict(idle=5), dict(seqs=3), dict(heads_first=True),
                                  dict(rope_rows=True), dict(odd_table=True), dict(packed=True, idle=2, rope_rows=True, heads_first=True)], ids=str)
def test_append_forms(mx, kind, more):
    check_append(mx, 2, kind, 23, 12, 4, 128, 16, 64, 2, **more)
    check_append(mx, 3, kind, 23, 12, 4, 64, 16, 64, 1, **more)


def test_append_without_sequence_numbers_and_saturation(mx):
    g = gen(5)
    cache = make_cache(mx, g, E4M3, 3, 20, 4, 2, 64)
    q, k, v = rand(g, 3, 4 * 64), rand(g, 3, 2 * 64), rand(g, 3, 2 * 64, std=1e4)
    v[1, 5] = float("nan")
    v[2, 7] = float("inf")
    pos = torch.tensor([0, 19, 7], device="cuda", dtype=torch.int32)
    q_out = torch.empty(3, 4, 64, device="cuda", dtype=torch.bfloat16)
    mx.qkv_norm_rope_append(q, k, v, 3, 4, 64, None, None, 1e-6, None, None, 0, 0, 0, cache, pos, q_out)
    assert torch.equal(q_out.view(3, -1), q)  # no norm, no rotation: a copy
    page = cache.page_table[torch.arange(3, device="cuda"), (pos // 4).long()].long()
    got = raw(cache.v)[page, (pos % 4).long()].view(torch.float8_e4m3fn).float()
    want = (v.float().view(3, 2, 64) / cache.v_scale[:, None])
    assert math.isnan(float(got[1, 0, 5])) and float(got[2, 0, 7]) == 448
    big = want.abs() > 470
    assert bool((got.abs()[big & want.isfinite()] == 448).all()) and int(big.sum()) > 100


@pytest.mark.parametrize("D, rot", [(64, 64), (128, 128), (80, 40), (48, 6)])
def test_append_e4m3_is_the_quotient_rounded_once(mx, D, rot):
    """v and, without a norm and with angles of zero, k: the code nearest to value / scale, of two that are equally near the even
    one, found by comparing the value with scale * (the middle between two codes), which is exact in 64 bits.  Scales of few bits
    have many quotients that lie in such a middle."""
    g = gen(7)
    scales = [7.0, 3.0, 5.0, 7 / 4096, 11 / 4096, 345 / 4096, 511 / 4096, 0.75]
    Hkv, T = len(scales), 1500
    k = torch.zeros(40, 50, Hkv, D, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    sc = torch.tensor(scales, device="cuda")
    cache = mx.KvCache(k, torch.zeros_like(k.view(torch.uint8)).view(torch.float8_e4m3fn), torch.randperm(40, device="cuda", generator=g).int()[None], sc, sc)
    # codes of the type in order, the middles between them, and values around those: exact ties where bf16 holds them
    code = torch.arange(127, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    middle = (code[1:] + code[:-1]) / 2
    pick = torch.randint(0, 126, (2, T, Hkv, D), device="cuda", generator=g)
    sign = torch.randint(0, 2, pick.shape, device="cuda", generator=g) * 2 - 1
    x = (sign * middle[pick] * sc.double()[:, None]).bfloat16()
    x[:, -100:] = rand(g, 2, 100, Hkv, D, std=30.0) * sc[:, None].bfloat16()
    q, pos = rand(g, T, D), torch.arange(T, device="cuda", dtype=torch.int32)
    angle = torch.zeros(T, rot // 2, device="cuda")
    mx.qkv_norm_rope_append(q, x[0], x[1], T, 1, D, None, None, 1e-6, angle.cos(), angle.sin(), T, rot, 2, cache, pos, torch.empty_like(q),
                            seq_ids=torch.zeros_like(pos))
    page, slot = cache.page_table[0].long()[pos.long() // 50], pos.long() % 50
    ties = 0
    for t, v in ((cache.k, x[0]), (cache.v, x[1])):
        a, s = v.double().abs(), sc.double()[:, None]
        below = (a[..., None] > s[..., None] * middle).sum(-1)  # middles below the value; one equal to it goes to the even code
        tie = (a[..., None] == s[..., None] * middle).any(-1)
        want = below + (tie & (below % 2 == 1))
        got = raw(t)[page, slot].long()
        assert torch.equal(got & 127, want) and torch.equal(got >> 7, torch.signbit(v).long())
        ties += int(tie.sum())
    assert ties > 100000  # the case that the test is about


def test_append_e4m3_scales_and_values_at_the_ends_of_fp32(mx):
    """Every bf16 number under scales from the smallest normal to the largest power of two: the fp32 quotient, rounded."""
    scales = torch.tensor([2.0 ** -126, 1.75 * 2.0 ** -126, 7 * 2.0 ** -100, 7 * 2.0 ** -64, 1.0, 7 * 2.0 ** 62, 7 * 2.0 ** 100, 1.75 * 2.0 ** 126,
                           2.0 ** 127, 1.75 * 2.0 ** 127])
    Hkv, D, T = len(scales), 64, 1024
    v = torch.arange(1 << 16, dtype=torch.int32).to(torch.uint16).view(torch.bfloat16).view(T, 1, D).expand(T, Hkv, D).contiguous()
    pages = torch.zeros(2, 16, 64, Hkv, D, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn)
    cache = mx.KvCache(pages[0], pages[1], torch.arange(16, device="cuda", dtype=torch.int32)[None], scales.cuda(), scales.cuda())
    q, pos, x = torch.zeros(T, D, device="cuda", dtype=torch.bfloat16), torch.arange(T, device="cuda", dtype=torch.int32), v.cuda()
    mx.qkv_norm_rope_append(q, x, x, T, 1, D, None, None, 1e-6, None, None, 0, 0, 0, cache, pos, torch.empty_like(q), seq_ids=torch.zeros_like(pos))
    want = (v.float() / scales[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    nan = v.isnan()
    for t in (cache.k, cache.v):
        got = raw(t).view(T, Hkv, D).cpu()
        assert torch.equal(got[~nan], want[~nan]) and bool(((got[nan] & 127) == 127).all())


def test_append_bad_indices_are_left_out_and_reported(mx):
    g = gen(6)
    cache = make_cache(mx, g, BF16, 6, 32, 16, 2, 64)
    cache.page_table[3, 1] = 99
    cache.page_table[4, 0] = -1
    before = cache.k.clone(), cache.v.clone()
    q, k, v = rand(g, 8, 4 * 64), rand(g, 8, 2 * 64), rand(g, 8, 2 * 64)
    ids = torch.tensor([0, 6, 2, 3, 4, 5, 1, 2**31 - 1], device="cuda", dtype=torch.int32)
    pos = torch.tensor([3, 0, 32, 16, 0, -1, 5, 2**31 - 1], device="cuda", dtype=torch.int32)
    q_out = torch.full((8, 4, 64), 7.0, device="cuda", dtype=torch.bfloat16)
    angle = torch.rand(5, 32, device="cuda")  # row 6 (position 5) lies behind the tables, row 0 (position 3) does not
    mx.qkv_norm_rope_append(q, k, v, 8, 4, 64, None, None, 1e-6, angle.cos(), angle.sin(), 5, 64, 2, cache, pos, q_out, seq_ids=ids)
    torch.cuda.synchronize()
    assert mx.device_error() == 2
    assert bool((q_out[1:] == 7).all()) and not bool((q_out[0] == 7).all())
    for t, old, x in ((cache.k, before[0], None), (cache.v, before[1], v)):
        page = int(cache.page_table[0, 0])
        if x is not None:
            assert torch.equal(t[page, 3].flatten(), x[0])
        t = t.clone()
        t[page, 3] = old[page, 3]
        assert torch.equal(raw(t), raw(old))


# ---- decode ---------------------------------------------------------------------------------------------------

def check_decode(mx, seed, kind, lens, H, Hkv, D, page, left=-1, sinks=0, heads_first=False, packed=False, scales=True, cache=None, q_std=1.0):
    g = gen(seed)
    n = len(lens)
    cache = cache or make_cache(mx, g, kind, n, max(max(lens), 1), page, Hkv, D, heads_first, scales=scales)
    buf = rand(g, n, H * D + (64 if packed else 0), std=q_std)
    q = buf[:, :H * D]
    out = torch.full((n, H, D), 7.0, device="cuda", dtype=torch.bfloat16)
    lse = torch.full((n, H), 7.0, device="cuda")
    ws = mx.attn_decode_workspace(cache, H)
    ws.fill_(255)  # NaN
    sl = torch.tensor(lens, device="cuda", dtype=torch.int32)
    mx.attn_decode_paged(q, cache, sl, H, D ** -0.5, out, left=left, sinks=sinks, q_stride=buf.stride(0), lse=lse, workspace=ws)
    want = R.decode_reference(q.reshape(n, H, D), cache, lens, H, D ** -0.5, left, sinks)
    R.assert_within(out, want[0], want[2], "out")
    R.assert_within(lse, want[1], want[3], "lse")
    again = torch.empty_like(out)
    mx.attn_decode_paged(q, cache, sl, H, D ** -0.5, again, left=left, sinks=sinks, q_stride=buf.stride(0), workspace=ws)
    assert torch.equal(again, out)


DECODE = [
    # lens, H, Hkv, D, page, left, sinks
    ([1], 1, 1, 128, 16, -1, 0), ([0], 2, 1, 64, 16, -1, 0), ([500], 32, 8, 128, 16, -1, 0), ([63, 64, 65, 0, 1, 129], 8, 2, 128, 16, -1, 0),
    ([0, 0, 5, 0], 4, 4, 64, 7, -1, 0), ([1000, 3, 777], 28, 4, 128, 100, -1, 0), ([300, 40], 16, 1, 96, 1, -1, 0),
    ([300, 40], 40, 1, 128, 24, -1, 0), ([257, 1, 64], 34, 2, 64, 64, -1, 0), ([2000], 8, 8, 80, 128, 100, 4),
    ([2000, 50, 101, 102, 105], 8, 2, 128, 16, 100, 4), ([2000, 5], 8, 2, 128, 16, 0, 0), ([2000, 5], 8, 2, 64, 16, 0, 1),
    ([2000, 700], 8, 2, 128, 16, 63, 1000), ([5000] * 3, 6, 3, 128, 256, 10 ** 12, 5), ([9000], 5, 5, 16, 32, -1, 0), ([130], 20, 4, 32, 16, -1, 0)]


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("case", DECODE, ids=str)
def test_decode(mx, kind, case):
    check_decode(mx, 11, kind, *case)


@pytest.mark.parametrize("D", [8, 24, 72, 104, 120])
def test_decode_bf16_head_sizes(mx, D):
    check_decode(mx, 12, BF16, [77, 200], 6, 2, D, 16)


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("more", [dict(heads_first=True), dict(packed=True), dict(scales=False), dict(q_std=30.0), dict(q_std=1e-6),
                                  dict(heads_first=True, packed=True)], ids=str)
def test_decode_forms(mx, kind, more):
    check_decode(mx, 13, kind, [333, 64, 1200, 2], 12, 4, 128, 48, **more)
    check_decode(mx, 14, kind, [333, 64, 1200, 2], 12, 4, 64, 48, left=200, sinks=3, **more)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_many_sequences(mx, kind):
    rng = random.Random(4)
    check_decode(mx, 15, kind, [rng.choice([0, 1, 5, 64, 100, rng.randrange(1, 400)]) for _ in range(300)], 4, 2, 64, 16)
    check_decode(mx, 16, kind, [rng.randrange(1, 3000) for _ in range(9)], 16, 2, 128, 64)


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_passes_over_many_empty_sequences(mx, kind):
    """A run of tiles that ends one sequence and goes on in the next one that has tokens, 200000 empty ones further: a wait between warps,
    here of 0.8 ms and what the sequences add to it, must not run out meanwhile."""
    g = gen(33)
    seqs, Hkv, D, page = 200000, 5, 128, 64
    cache = make_cache(mx, g, kind, 2, 4224, page, Hkv, D)
    table = torch.full((seqs, 70), -1, dtype=torch.int32, device="cuda")
    table[0, :66], table[-1, :66] = cache.page_table[0], cache.page_table[1]
    wide = mx.KvCache(cache.k, cache.v, table, cache.k_scale, cache.v_scale)
    q = rand(g, seqs, Hkv * D).view(seqs, Hkv, D)
    mx.set_tuning("decode_wait_tries", 1 << 9)
    try:
        for first in (61 * 64, 62 * 64 - 3, 63 * 64):
            lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
            lens[0], lens[-1] = first, 4160
            out, lse = torch.full_like(q, 7.0), torch.full((seqs, Hkv), 7.0, device="cuda")
            mx.attn_decode_paged(q, wide, lens, Hkv, D ** -0.5, out, lse=lse, workspace=mx.attn_decode_workspace(wide, Hkv))
            want = R.decode_reference(q[[0, -1]], cache, [first, 4160], Hkv, D ** -0.5, -1, 0)
            R.assert_within(out[[0, -1]], want[0], want[2])
            R.assert_within(lse[[0, -1]], want[1], want[3])
            assert not bool(out[1:-1].any()) and bool((lse[1:-1] == -math.inf).all())
    finally:
        mx.set_tuning("decode_wait_tries", 0)


def test_decode_uneven_scores(mx):
    """A key whose score lies far above all others, late in the sequence: what was summed before it has to vanish."""
    g = gen(17)
    cache = make_cache(mx, g, BF16, 2, 700, 16, 1, 128)
    q = rand(g, 2, 4, 128)
    for b in range(2):
        page, slot = int(cache.page_table[b, 650 // 16]), 650 % 16
        cache.k[page, slot, 0] = q[b, 1] * 40
    out, lse = torch.empty(2, 4, 128, device="cuda", dtype=torch.bfloat16), torch.empty(2, 4, device="cuda")
    mx.attn_decode_paged(q, cache, torch.tensor([700, 651], device="cuda", dtype=torch.int32), 4, 128 ** -0.5, out, lse=lse,
                         workspace=mx.attn_decode_workspace(cache, 4))
    want = R.decode_reference(q, cache, [700, 651], 4, 128 ** -0.5, -1, 0)
    R.assert_within(out, want[0], want[2])
    R.assert_within(lse, want[1], want[3])


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_reads_nothing_out_of_view(mx, kind):
    """NaN in every cached token that is out of view, behind the length and in pages of nobody: the same output."""
    g = gen(18)
    lens, left, sinks = [500, 130, 64, 0], 100, 5
    cache = make_cache(mx, g, kind, 4, 512, 24, 2, 128)
    q = rand(g, 4, 8, 128)
    sl = torch.tensor(lens, device="cuda", dtype=torch.int32)
    ws = mx.attn_decode_workspace(cache, 8)
    outs = []
    for poison in (False, True):
        if poison:
            keep = torch.zeros(cache.k.shape[:2], dtype=torch.bool, device="cuda")
            for b, n in enumerate(lens):
                j = torch.arange(n, device="cuda")
                j = j[(j >= n - 1 - left) | (j < sinks)]
                keep[cache.page_table[b].long()[j // 24], j % 24] = True
            for t in (cache.k, cache.v):
                raw(t)[~keep] = 0x7F if kind == E4M3 else 0x7FC0
        out = torch.empty(4, 8, 128, device="cuda", dtype=torch.bfloat16)
        mx.attn_decode_paged(q, cache, sl, 8, 0.1, out, left=left, sinks=sinks, workspace=ws)
        outs.append(out)
    assert bool(torch.isfinite(outs[0]).all()) and torch.equal(outs[0], outs[1])


def test_decode_nan_in_view_stays_in_its_sequence(mx):
    g = gen(19)
    cache = make_cache(mx, g, BF16, 3, 200, 16, 2, 64)
    cache.v[int(cache.page_table[1, 2]), 3, 1, 5] = float("nan")
    q, out, lse = rand(g, 3, 4, 64), torch.empty(3, 4, 64, device="cuda", dtype=torch.bfloat16), torch.empty(3, 4, device="cuda")
    mx.attn_decode_paged(q, cache, torch.tensor([200, 150, 180], device="cuda", dtype=torch.int32), 4, 0.125, out, lse=lse,
                         workspace=mx.attn_decode_workspace(cache, 4))
    nan = out.isnan()
    assert bool(nan[1, 2:, 5].all()) and int(nan.sum()) == 2 and bool(lse.isfinite().all())


def test_decode_bad_pages_and_lengths_are_left_out_and_reported(mx):
    g = gen(20)
    cache = make_cache(mx, g, BF16, 4, 64, 16, 1, 64)
    q = rand(g, 4, 2, 64)
    ws = mx.attn_decode_workspace(cache, 2)
    good = torch.empty(4, 2, 64, device="cuda", dtype=torch.bfloat16)
    mx.attn_decode_paged(q, cache, torch.tensor([64, 60, 0, 64], device="cuda", dtype=torch.int32), 2, 0.125, good, workspace=ws)
    torch.cuda.synchronize()
    assert mx.device_error() == 0
    out = torch.empty_like(good)
    # a length past the table: the table's tokens; a negative one: none
    mx.attn_decode_paged(q, cache, torch.tensor([1 << 30, 60, -7, 64], device="cuda", dtype=torch.int32), 2, 0.125, out, workspace=ws)
    torch.cuda.synchronize()
    assert mx.device_error() == 2
    assert torch.equal(out, good)
    # pages out of range: their tokens are left out
    cache.page_table[1, 1] = cache.k.shape[0]
    cache.page_table[3, 0] = -5
    mx.attn_decode_paged(q, cache, torch.tensor([64, 60, 0, 16], device="cuda", dtype=torch.int32), 2, 0.125, out, workspace=ws)
    torch.cuda.synchronize()
    assert mx.device_error() == 2
    k, v = (torch.cat([R.gather(t, cache.page_table[1, [0, 2, 3]], 44)]) for t in (cache.k, cache.v))
    want = [R.attention_rows(q[1, h][None], k[:, 0], v[:, 0], 0.125, R.visible(1, 44, -1, 0, 0, "cuda")) for h in range(2)]
    for h in range(2):
        R.assert_within(out[1, h][None], want[h][0], want[h][2])
    assert bool((out[3] == 0).all()) and torch.equal(out[0], good[0])


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_without_a_page(mx, kind):
    """A cache of no pages at all: every token is left out and reported, whatever the table says."""
    empty = torch.zeros(2, 0, 16, 2, 64, device="cuda", dtype=torch.bfloat16 if kind == BF16 else torch.uint8)
    empty = empty if kind == BF16 else empty.view(torch.float8_e4m3fn)
    cache = mx.KvCache(empty[0], empty[1], torch.tensor([[0, 1], [-1, 5]], device="cuda", dtype=torch.int32))
    q, lse = rand(gen(30), 2, 4, 64), torch.full((2, 4), 7.0, device="cuda")
    out = torch.full_like(q, 7.0)
    mx.attn_decode_paged(q, cache, torch.tensor([20, 32], device="cuda", dtype=torch.int32), 4, 0.125, out, lse=lse, workspace=mx.attn_decode_workspace(cache, 4))
    torch.cuda.synchronize()
    assert mx.device_error() == 2
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_decode_refuses_a_small_workspace(mx):
    g = gen(24)
    cache = make_cache(mx, g, BF16, 2, 4000, 16, 2, 128)
    q, out = rand(g, 2, 8, 128), torch.full((2, 8, 128), 7.0, device="cuda", dtype=torch.bfloat16)
    sl = torch.tensor([4000, 100], device="cuda", dtype=torch.int32)
    with pytest.raises(mx.MxkError, match="workspace"):
        mx.attn_decode_paged(q, cache, sl, 8, 0.09, out, workspace=mx.attn_decode_workspace(cache, 8)[:4096])
    torch.cuda.synchronize()
    assert bool((out == 7).all())


def test_decode_rows_of_more_than_31_bits(mx):
    """More than 2^31 elements in the heads of one sequence: none of them left out where it is empty, and all of them right where it
    has one token (its value, whatever the query)."""
    H, D = (1 << 24) + 3, 128
    kv = rand(gen(32), 2, 1, 16, 1, D)
    cache = mx.KvCache(kv[0], kv[1], torch.zeros(2, 1, dtype=torch.int32, device="cuda"))
    q = torch.zeros(H, D, device="cuda", dtype=torch.bfloat16)
    out, lse = torch.full((2, H, D), 7.0, device="cuda", dtype=torch.bfloat16), torch.full((2, H), 7.0, device="cuda")
    mx.attn_decode_paged(q, cache, torch.tensor([0, 1], device="cuda", dtype=torch.int32), H, 0.1, out, q_stride=0, lse=lse, workspace=mx.attn_decode_workspace(cache, H))
    assert not bool(out[0].view(torch.int64).any()) and bool((lse[0] == -math.inf).all())
    assert torch.equal(out[1], kv[1, 0, 0].expand(H, D)) and not bool(lse[1].any())
    del q, out, lse
    torch.cuda.empty_cache()


def test_decode_offsets_past_32_bits(mx):
    g = gen(21)
    pages, page, Hkv, D = 18000, 128, 8, 128  # 2.36e9 elements each
    k = torch.zeros(pages, page, Hkv, D, device="cuda", dtype=torch.bfloat16)
    v = torch.zeros_like(k)
    far = torch.arange(pages - 6, pages, device="cuda")
    k[far], v[far] = rand(g, 6, page, Hkv, D), rand(g, 6, page, Hkv, D)
    cache = mx.KvCache(k, v, far.view(2, 3).to(torch.int32))
    check_decode(mx, 22, BF16, [384, 200], 8, 8, 128, page, cache=cache)
    del k, v, cache
    torch.cuda.empty_cache()


def test_decode_the_longest_sequence(mx):
    """2^31 - 2 tokens, all but the last few in one page that the table names again and again: keys of zero and values of one, so that
    every sum is a whole number of 2^7 below 2^24 of them in a run, and fp32 holds it; the second sequence ends in a page whose
    last key outweighs all others (e^40 against 2^31 < e^22)."""
    page, pages, D = 32767, 65538, 16
    kv = torch.zeros(2, 2, page, 1, D, device="cuda")
    kv[1] = 1.0
    kv[0, 1, -1], kv[1, 1, -1] = 2.5, -2.0
    kv = kv.to(torch.float8_e4m3fn)
    table = torch.zeros(2, pages, dtype=torch.int32, device="cuda")
    table[1, -1] = 1
    cache = mx.KvCache(kv[0], kv[1], table)
    n = page * pages
    assert n == 2 ** 31 - 2
    q, lens = torch.ones(2, 1, D, device="cuda", dtype=torch.bfloat16), torch.full((2,), n, dtype=torch.int32, device="cuda")
    ws = mx.attn_decode_workspace(cache, 1)
    for left, sinks in ((-1, 0), (n - 2, 1), (1000, 3)):
        out, lse = torch.full_like(q, 7.0), torch.full((2, 1), 7.0, device="cuda")
        mx.attn_decode_paged(q, cache, lens, 1, 1.0, out, left=left, sinks=sinks, lse=lse, workspace=ws)
        seen = n if left < 0 else min(n, left + 1 + sinks)
        assert bool((out[0] == 1).all()) and bool((out[1] == -2).all())
        want = torch.tensor([math.log(seen), 40 + math.log1p(seen * math.exp(-40))])
        assert float((lse.cpu()[:, 0].double() - want).abs().max()) <= 2.0 ** -18  # steps of 2^-22 near 21 and 40, log2 and exp2 to 2^-22


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_many_small_weights(mx, kind):
    """A million tokens of weight 2^-25.1 behind one of weight 1, as many work items as fill the GPU with such runs: what the
    small ones add up to must not be lost in the type that the product with V takes them in."""
    seqs, Hkv, D, page, pages = 64, 8, 64, 64, 16384
    L, bits = page * pages, 25.1
    k, v = torch.full((2, page, Hkv, D), -1.0, device="cuda"), torch.full((2, page, Hkv, D), 448.0, device="cuda")
    k[0, 0], v[0, 0] = 0.0, 2.0 ** -4
    dtype = torch.bfloat16 if kind == BF16 else torch.float8_e4m3fn
    table = torch.ones(seqs, pages, dtype=torch.int32, device="cuda")
    table[:, 0] = 0
    cache = mx.KvCache(k.to(dtype), v.to(dtype), table)
    q = torch.ones(seqs, Hkv, D, dtype=torch.bfloat16, device="cuda")
    out, lse = torch.empty_like(q), torch.empty(seqs, Hkv, device="cuda")
    lens = torch.full((seqs,), L, dtype=torch.int32, device="cuda")
    mx.attn_decode_paged(q, cache, lens, Hkv, bits * math.log(2) / D, out, lse=lse, workspace=mx.attn_decode_workspace(cache, Hkv))
    small = (L - 1) * 2.0 ** -bits
    want = (2.0 ** -4 + small * 448) / (1 + small)
    # fp32 sums over a run: one step of 2^-23 for each of its L / 16 products, of the output's largest partial sum, which is
    # the output; a thread's sum of weights takes one step of 2^-23 for each of its L / 64 tiles
    steps = L / 16 * 2.0 ** -23
    assert (out.double() - want).abs().max().item() <= want * (2.0 ** -8 + 2.0 ** -8 + 2 * steps)
    assert (lse.double() - math.log1p(small)).abs().max().item() <= L / 64 * 2.0 ** -23 + 2.0 ** -20


def test_decode_in_a_graph_on_another_stream(mx):
    """Captured once, replayed with other lengths, queries and tables: the call reads all of them on the device."""
    g = gen(23)
    cache = make_cache(mx, g, BF16, 3, 400, 16, 2, 128)
    q, sl = rand(g, 3, 8, 128), torch.tensor([400, 17, 0], device="cuda", dtype=torch.int32)
    out, lse = torch.empty(3, 8, 128, device="cuda", dtype=torch.bfloat16), torch.empty(3, 8, device="cuda")
    ws = mx.attn_decode_workspace(cache, 8)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        mx.attn_decode_paged(q, cache, sl, 8, 0.09, out, lse=lse, workspace=ws, stream=torch.cuda.current_stream())
    for lens in ([400, 17, 0], [1, 400, 300], [0, 0, 0], [399, 64, 65]):
        sl.copy_(torch.tensor(lens, dtype=torch.int32))
        q.copy_(rand(g, 3, 8, 128))
        cache.page_table.copy_(cache.page_table.flip(0))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        want = R.decode_reference(q, cache, lens, 8, 0.09, -1, 0)
        R.assert_within(out, want[0], want[2])
        R.assert_within(lse, want[1], want[3])


# ---- window ---------------------------------------------------------------------------------------------------

def check_window(mx, seed, rows, keys, H, Hkv, D, left=-1, right=-1, sinks=0, packed=False, behind=0, cu=True, std=1.0, scale=None,
                 edit=None, pad_out=0, lse=True):
    g = gen(seed)
    nq, nk = sum(rows) + behind, sum(keys) + behind
    scale = scale or D ** -0.5
    if packed:
        buf = rand(g, nq, (H + 2 * Hkv) * D, std=std)
        q, k, v = buf[:, :H * D], buf[:, H * D:(H + Hkv) * D], buf[:, (H + Hkv) * D:]
    else:
        q, k, v = rand(g, nq, H * D, std=std), rand(g, nk, Hkv * D, std=std), rand(g, nk, Hkv * D)
    if edit:
        edit(q.view(nq, H, D) if not packed else q.unflatten(1, (H, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, D)))
    full = torch.full((nq, H * D + pad_out), 7.0, device="cuda", dtype=torch.bfloat16)
    ls = torch.full((nq, H), 7.0, device="cuda") if lse else None
    ends = [torch.tensor([sum(n[:i]) for i in range(len(n) + 1)], device="cuda", dtype=torch.int32) for n in (rows, keys)] if cu else [None, None]
    mx.attn_window(q, k, v, nq, nk, H, Hkv, D, scale, full, left=left, right=right, sinks=sinks, cu_q=ends[0], cu_k=ends[1], q_stride=q.stride(0),
                   k_stride=k.stride(0), v_stride=v.stride(0), out_stride=full.stride(0), lse=ls)
    out = full[:, :H * D].unflatten(1, (H, D))
    want = R.window_reference(q.unflatten(1, (H, D)), k.unflatten(1, (Hkv, D)), v.unflatten(1, (Hkv, D)), rows, keys, H, Hkv, D, scale, left, right,
                              sinks)
    n = sum(rows)
    R.assert_within(out[:n], want[0][:n], want[2][:n], "out")
    if lse:
        R.assert_within(ls[:n], want[1][:n], want[3][:n], "lse")
        assert bool((ls[n:] == 7).all())
    assert bool((full[n:] == 7).all()) and bool((full[:, H * D:] == 7).all())
    return out, ls


WINDOW = [
    # rows, keys, H, Hkv, D, left, right, sinks
    ([1], [1], 1, 1, 128, -1, -1, 0), ([1], [300], 4, 2, 64, -1, 0, 0), ([77], [77], 8, 2, 128, -1, 0, 0), ([128], [128], 2, 2, 128, -1, -1, 0),
    ([129], [129], 2, 1, 128, -1, 0, 0), ([256], [256], 3, 3, 64, -1, 0, 0), ([257], [513], 2, 2, 128, -1, -1, 0), ([255], [383], 2, 2, 128, -1, 0, 0),
    ([700], [700], 2, 2, 128, 128, 0, 4), ([700], [700], 2, 2, 128, 127, 129, 130), ([700], [700], 2, 2, 64, 0, 0, 0), ([700], [700], 1, 1, 128, 5, -1, 1),
    ([700], [700], 1, 1, 128, 0, 0, 1), ([1000], [1000], 1, 1, 128, 200, 100, 500), ([300], [40], 2, 1, 128, -1, 0, 0), ([300], [40], 2, 1, 128, 3, 2, 1),
    ([300], [40], 2, 1, 64, -1, -1, 0), ([50], [0], 2, 1, 128, -1, -1, 0), ([5, 0, 300, 1, 128, 17], [5, 3, 310, 1, 128, 17], 4, 2, 128, -1, 0, 0),
    ([5, 0, 300, 1, 128, 17], [0, 3, 310, 2, 100, 170], 4, 2, 64, 60, 30, 2), ([2000, 30], [2000, 30], 2, 1, 128, -1, -1, 0),
    ([513] * 3, [513] * 3, 5, 5, 72, -1, -1, 0), ([100, 200], [150, 250], 6, 3, 8, -1, 0, 0), ([300], [300], 2, 2, 80, 50, 0, 3),
    ([300], [300], 2, 2, 120, -1, 0, 0), ([300], [300], 2, 1, 32, -1, 50, 0), ([1], [5000], 2, 1, 128, 1000, 0, 10), ([900], [3000], 1, 1, 128, 1000, 0, 10)]


@pytest.mark.parametrize("case", WINDOW, ids=str)
def test_window(mx, case):
    check_window(mx, 31, *case)


@pytest.mark.parametrize("more", [dict(packed=True), dict(behind=37), dict(cu=False), dict(std=4.0), dict(std=0.01), dict(pad_out=64), dict(lse=False),
                                  dict(packed=True, behind=200), dict(scale=1.0)], ids=str)
def test_window_forms(mx, more):
    check_window(mx, 32, [333], [333], 6, 2, 128, -1, 0, 0, **more)
    check_window(mx, 33, [333], [333], 6, 2, 64, 100, 20, 7, **more)
    if more.get("cu", True):
        check_window(mx, 34, [130, 3, 400], [130, 3, 400], 4, 4, 128, 64, 0, 2, **more)


def test_window_many_sequences(mx):
    rng = random.Random(8)
    rows = [rng.choice([0, 1, 2, rng.randrange(1, 200)]) for _ in range(150)]
    check_window(mx, 35, rows, [n + rng.randrange(0, 30) for n in rows], 2, 1, 64, -1, 0, 0)


def test_window_thousands_of_sequences(mx):
    """More sequences than a search looks at at once, most of them empty or of one row."""
    rng = random.Random(9)
    rows = [rng.choice([0, 0, 1, 1, 2, 5]) for _ in range(1500)]
    rows[3], rows[700], rows[1499] = 300, 129, 257
    check_window(mx, 36, rows, [n + (i % 3 if n else 0) for i, n in enumerate(rows)], 1, 1, 64, -1, 0, 0)
    check_window(mx, 36, [1] * 700, [1] * 700, 2, 1, 128, 3, 0, 1, behind=5)


@pytest.fixture(params=[1, 2], ids=["from_the_back", "from_the_front"])
def order(mx, request):
    mx.set_tuning("window_order", request.param)
    yield request.param
    mx.set_tuning("window_order", 0)


def test_window_tiles_in_either_order(mx, order):
    """Many more tiles than CTAs at a time, looked for in rising and in falling order, with searches past the first sequences and
    numbers that no tile has: every row is computed once whatever order the tiles come in."""
    rng = random.Random(10)
    rows = [rng.choice([0, 1, 3, 40, 129, 300]) for _ in range(400)]
    check_window(mx, 51, rows, rows, 4, 2, 64, -1, 0, 0, behind=9)
    check_window(mx, 52, [1] * 900, [2] * 900, 2, 1, 128, 3, 0, 1)
    check_window(mx, 53, [9000], [9000], 8, 2, 64, 200, 0, 3, cu=False)


@pytest.mark.parametrize("left, right, sinks", [(-1, -1, 0), (-1, 0, 0), (300, 0, 5), (400, 150, 130)])
@pytest.mark.parametrize("D", [128, 64])
def test_window_second_tiles(mx, order, D, left, right, sinks):
    """More tiles than the GPU has CTAs for, of two halves and several blocks each, so that a CTA goes from one to the next: the ring of
    stages and the queries used again, the next tile's scores under the last one's output."""
    check_window(mx, 56, [1500, 900, 1211], [1500, 1300, 1211], 24, 8, D, left, right, sinks, behind=3)


def test_window_scores_that_grow_along_the_keys(mx):
    """Every block of keys has a larger maximum than the one in front of it, by more and by less than a factor of 2^8."""
    def edit(q, k, v):
        q[:] = q.abs()
        k[:] = k.abs() * torch.linspace(0.01, 6, k.shape[0], device="cuda").bfloat16()[:, None, None]
    check_window(mx, 36, [400], [2000], 2, 1, 128, edit=edit)
    check_window(mx, 37, [900], [900], 2, 1, 64, -1, 0, 0, edit=edit, scale=1.0)
    check_window(mx, 38, [900], [900], 2, 1, 128, -1, 0, 0, edit=lambda q, k, v: k.mul_(torch.linspace(20, 0.1, 900, device="cuda").bfloat16()[:, None, None]))


def test_window_rows_of_nobody_may_hold_anything(mx):
    """NaN and infinities in rows behind the last sequence and in keys that no row sees."""
    def edit(q, k, v):
        q[400:] = float("nan")
        k[400:], v[400:] = float("nan"), float("inf")
    check_window(mx, 39, [150, 250], [150, 250], 2, 2, 128, -1, 0, 0, behind=60, edit=edit)
    check_window(mx, 40, [150, 250], [150, 250], 2, 2, 64, -1, -1, 0, behind=1, edit=edit)

    def unseen(q, k, v):  # a window over the last keys of a long prefix: keys 10 .. 500 are nobody's
        k[10:500], v[10:500] = float("nan"), float("-inf")
    check_window(mx, 41, [100], [700], 2, 1, 128, 99, 0, 10, edit=unseen)


def test_window_rows_taken_again_outlast_a_wait(mx):
    """Values behind the last key that are not finite: every row is taken again by a loop over its keys, 20 ms a tile, and the CTAs'
    next tiles stand behind that.  A wait between warps, here of 3 ms and what the keys add to it, must not run out meanwhile."""
    def edit(q, k, v):
        k[4000:], v[4000:] = float("nan"), float("inf")
    mx.set_tuning("window_wait_tries", 1 << 11)
    try:
        check_window(mx, 54, [64], [4000], 160, 1, 64, behind=20, edit=edit)
        check_window(mx, 55, [33, 31], [2000, 4000 - 2000], 90, 2, 128, behind=1, edit=edit)
    finally:
        mx.set_tuning("window_wait_tries", 0)


@pytest.mark.parametrize("what", ["nan", "inf"])
def test_window_values_reach_only_rows_that_see_them(mx, what):
    """A NaN or an infinity in the values of one key: rows that do not see the key are as they would be without it."""
    bad = float(what)
    rows, H, D = 400, 2, 128
    for left, right, sinks, key in ((-1, 0, 0, 200), (60, 0, 0, 150), (60, 0, 3, 1), (50, 50, 0, 255), (-1, 0, 0, 399), (10, -1, 0, 130)):
        g = gen(42)
        q, k, v = (rand(g, rows, H * D) for _ in range(3))
        outs = []
        for poison in (False, True):
            if poison:
                v[key, 5] = bad
            out = torch.empty(rows, H, D, device="cuda", dtype=torch.bfloat16)
            mx.attn_window(q, k, v, rows, rows, H, H, D, 0.088, out, left=left, right=right, sinks=sinks)
            outs.append(out)
        sees = R.visible(rows, rows, left, right, sinks, "cuda")[:, key]
        hit = torch.zeros_like(outs[1], dtype=torch.bool)
        hit[sees, 0, 5] = True
        got = outs[1][hit]
        assert bool((got.isnan() if what == "nan" else got.isnan() | (got == bad)).all())
        ok = ~hit
        assert bool(outs[1][ok].isfinite().all())
        err = (outs[1][ok].double() - outs[0][ok].double()).abs()
        assert float((err - 2.0 ** -6 * outs[0][ok].double().abs() - 2.0 ** -7).max()) <= 0  # two bf16 roundings each of values of size one


def test_window_bad_sequence_ends_are_reported(mx):
    g = gen(43)
    q, k, v = rand(g, 100, 128), rand(g, 100, 128), rand(g, 100, 128)
    out = torch.empty(100, 1, 128, device="cuda", dtype=torch.bfloat16)
    for cq, ck in (([0, 50, 400], [0, 50, 100]), ([0, 50, 100], [0, 70, 1000]), ([0, 50, 100], [0, -5, 90]), ([0, 60, 40], [0, 50, 100]),
                   ([-3, 50, 100], [0, 50, 100])):
        cu = [torch.tensor(t, device="cuda", dtype=torch.int32) for t in (cq, ck)]
        mx.attn_window(q, k, v, 100, 100, 1, 1, 128, 0.09, out, right=0, cu_q=cu[0], cu_k=cu[1])
        torch.cuda.synchronize()
        assert mx.device_error() == 2, (cq, ck)


def test_window_offsets_past_32_bits(mx):
    g = gen(44)
    rows, stride = 600, 4 << 20  # rows 8 MiB apart: 2.5e9 elements
    buf = torch.empty(rows * stride, device="cuda", dtype=torch.bfloat16)
    wide = buf.view(rows, stride)
    q, k, v = wide[:, :256], wide[:, 256:512], wide[:, 512:768]
    for t in (q, k, v):
        t.copy_(rand(g, rows, 256))
    out = torch.empty(rows, 2, 128, device="cuda", dtype=torch.bfloat16)
    mx.attn_window(q, k, v, rows, rows, 2, 2, 128, 0.088, out, right=0, q_stride=stride, k_stride=stride, v_stride=stride)
    want = R.window_reference(*(t.unflatten(1, (2, 128)) for t in (q, k, v)), [rows], [rows], 2, 2, 128, 0.088, -1, 0, 0)
    R.assert_within(out, want[0], want[2])
    del buf, wide, q, k, v
    torch.cuda.empty_cache()


def test_window_in_a_graph_on_another_stream(mx):
    g = gen(45)
    q, k, v = rand(g, 300, 256), rand(g, 300, 128), rand(g, 300, 128)
    cu = torch.tensor([0, 100, 300], device="cuda", dtype=torch.int32)
    out = torch.empty(300, 2, 128, device="cuda", dtype=torch.bfloat16)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
        mx.attn_window(q, k, v, 300, 300, 2, 1, 128, 0.088, out, right=0, cu_q=cu, cu_k=cu, stream=torch.cuda.current_stream())
    for ends in ([0, 100, 300], [0, 1, 300], [0, 0, 257]):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        q.copy_(rand(g, 300, 256))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        n = [b - a for a, b in zip(ends, ends[1:])]
        want = R.window_reference(q.view(300, 2, 128), k.view(300, 1, 128), v.view(300, 1, 128), n, n, 2, 1, 128, 0.088, -1, 0, 0)
        R.assert_within(out[:ends[-1]], want[0][:ends[-1]], want[2][:ends[-1]])


# ---- together -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_a_prompt_and_then_single_tokens(mx, kind):
    """A prompt through append + attn_window, then tokens one at a time through append + attn_decode_paged: each step equals
    the last row of a causal attention over everything so far."""
    g = gen(50)
    H, Hkv, D, page, left, sinks = 8, 2, 128, 16, 70, 4
    prompt, steps = [100, 37, 1], 5
    n, most = len(prompt), max(prompt) + steps
    cache = make_cache(mx, g, kind, n, most, page, Hkv, D, fill=False)
    if kind == E4M3:
        cache.k_scale.fill_(0.02), cache.v_scale.fill_(0.02)
    wq, wk = 1 + 0.1 * torch.randn(D, device="cuda", generator=g), 1 + 0.1 * torch.randn(D, device="cuda", generator=g)
    angle = torch.arange(most, device="cuda")[:, None] * 1000.0 ** (-torch.arange(D // 2, device="cuda") / (D // 2))
    cos, sin = angle.cos(), angle.sin()
    stride = (H + 2 * Hkv) * D
    ws = mx.attn_decode_workspace(cache, H)

    def append(qkv, ids, pos, q_out, k_out=None):
        mx.qkv_norm_rope_append(qkv, qkv[:, H * D:], qkv[:, (H + Hkv) * D:], qkv.shape[0], H, D, wq, wk, 1e-6, cos, sin, most, D, 2, cache, pos, q_out,
                                seq_ids=ids, k_out=k_out, q_stride=stride, k_stride=stride, v_stride=stride)

    T = sum(prompt)
    qkv = rand(g, T, stride)
    ids = torch.repeat_interleave(torch.arange(n), torch.tensor(prompt)).int().cuda()
    pos = torch.cat([torch.arange(m) for m in prompt]).int().cuda()
    cu = torch.tensor([0, 100, 137, 138], device="cuda", dtype=torch.int32)
    q_out, k_out = torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16), torch.empty(T, Hkv, D, device="cuda", dtype=torch.bfloat16)
    append(qkv, ids, pos, q_out, k_out)
    out = torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16)
    v = qkv[:, (H + Hkv) * D:]
    mx.attn_window(q_out, k_out, v, T, T, H, Hkv, D, D ** -0.5, out, left=left, right=0, sinks=sinks, cu_q=cu, cu_k=cu, v_stride=stride)
    want = R.window_reference(q_out, k_out, v.unflatten(1, (Hkv, D)), prompt, prompt, H, Hkv, D, D ** -0.5, left, 0, sinks)
    R.assert_within(out, want[0], want[2])
    keys = [list(k_out[cu[b]:cu[b + 1]]) for b in range(n)]
    vals = [list(v.unflatten(1, (Hkv, D))[cu[b]:cu[b + 1]]) for b in range(n)]
    lens = torch.tensor(prompt, device="cuda", dtype=torch.int32)
    for _ in range(steps):
        qkv = rand(g, n, stride)
        q1, k1, o1 = (torch.empty(n, h, D, device="cuda", dtype=torch.bfloat16) for h in (H, Hkv, H))
        append(qkv, None, lens, q1, k1)
        lens += 1
        mx.attn_decode_paged(q1, cache, lens, H, D ** -0.5, o1, left=left, sinks=sinks, workspace=ws)
        ln = lens.tolist()
        want = R.decode_reference(q1, cache, ln, H, D ** -0.5, left, sinks)
        R.assert_within(o1, want[0], want[2])
        for b in range(n):
            keys[b].append(k1[b]), vals[b].append(qkv[b, (H + Hkv) * D:].view(Hkv, D))
            ref = R.window_reference(q1[b][None], torch.stack(keys[b]), torch.stack(vals[b]), [1], [ln[b]], H, Hkv, D, D ** -0.5, left, 0, sinks)
            if kind == BF16:  # the cache holds what k_out and v hold
                R.assert_within(o1[b][None], ref[0], ref[2])
            else:  # e4m3: each k and v off by 2^-4 of itself at most (and 2^-10 steps), a score by 2^-4 of its products
                size = D ** -0.5 * (q1[b].float().abs().view(H, D).amax(1) * torch.stack(keys[b]).float().abs().sum(-1).amax())
                assert bool(((o1[b].double() - ref[0][0]).norm(dim=1) <= ref[0][0].norm(dim=1) + 4).all()) and bool(size.isfinite().all())


def test_single_tokens_over_8_bits_against_what_went_in(mx):
    """Append into an e4m3 cache and attention over it, against a softmax in 64 bits of the very inputs.  Bounds: a stored key is off by at
    most 2^-4 of itself and 2^-10 scales (half a step, normal and subnormal), q_out by 2^-8, so a score by d = scale * sum(|q| dk +
    dq (|k| + dk)), a weight by a factor exp(2 d), and the output by (exp(2 d) - 1) sum w |v| + exp(2 d) sum w dv and the kernel's own
    roundings.  Queries, keys and values of one sign make the scores and outputs many times as large as that: an output of
    zero, or of another scale, fails."""
    g = gen(57)
    H, Hkv, D, page, left, sinks, steps, ks, vs = 8, 2, 128, 16, 70, 4, 5, 0.02, 0.013
    start = [100, 37, 1]
    n, most = len(start), max(start) + steps
    cache = make_cache(mx, g, E4M3, n, most, page, Hkv, D, fill=False)
    cache.k_scale.fill_(ks), cache.v_scale.fill_(vs)
    wq, wk = 0.2 + 0.02 * torch.rand(D, device="cuda", generator=g), 1 + 0.1 * torch.rand(D, device="cuda", generator=g)
    ws, scale = mx.attn_decode_workspace(cache, H), D ** -0.5
    keys, vals = [[] for _ in range(n)], [[] for _ in range(n)]

    def append(ids, pos):
        T = len(ids)
        q, k = rand(g, T, H, D).abs() + 0.01, rand(g, T, Hkv, D).abs() + 0.01
        v, q_out = (1 + 0.3 * rand(g, T, Hkv, D)).bfloat16(), torch.empty(T, H, D, device="cuda", dtype=torch.bfloat16)
        mx.qkv_norm_rope_append(q, k, v, T, H, D, wq, wk, 1e-6, None, None, 0, 0, 0, cache, torch.tensor(pos, dtype=torch.int32).cuda(), q_out,
                                seq_ids=torch.tensor(ids, dtype=torch.int32).cuda())
        k64 = R.rope_reference(k, wk, None, None, 0, 0, 1e-6)
        for t, b in enumerate(ids):
            keys[b].append(k64[t]), vals[b].append(v[t].double())
        return q_out, R.rope_reference(q, wq, None, None, 0, 0, 1e-6)

    append([b for b in range(n) for _ in range(start[b])], [t for b in range(n) for t in range(start[b])])
    for i in range(steps):
        lens = [m + i + 1 for m in start]
        q_out, q64 = append(list(range(n)), [m + i for m in start])
        out, lse = torch.empty_like(q_out), torch.empty(n, H, device="cuda")
        mx.attn_decode_paged(q_out, cache, torch.tensor(lens, dtype=torch.int32).cuda(), H, scale, out, left=left, sinks=sinks, lse=lse, workspace=ws)
        own = R.decode_reference(q_out, cache, lens, H, scale, left, sinks)
        for b, m in enumerate(lens):
            see = R.visible(1, m, left, 0, sinks, "cuda")[0]
            for h in range(H):
                q, k, v = q64[b, h], torch.stack(keys[b])[see, h * Hkv // H], torch.stack(vals[b])[see, h * Hkv // H]
                s = scale * k @ q
                w = s.softmax(0)
                dk, dv, dq = (2.0 ** -4 + 2.0 ** -16) * k + 2.0 ** -10 * ks, 2.0 ** -4 * v.abs() + 2.0 ** -10 * vs, (2.0 ** -8 + 2.0 ** -16) * q
                d = float((scale * (dk @ q + (k + dk) @ dq)).max())
                bound = math.expm1(2 * d) * (w @ v.abs()) + math.exp(2 * d) * (w @ dv) + own[2][b, h]
                want, want_lse = w @ v, torch.logsumexp(s, 0)
                assert bool(((out[b, h].double() - want).abs() <= bound).all())
                assert abs(float(lse[b, h].double() - want_lse)) <= d + float(own[3][b, h])
                # what the bounds would refuse: an output of zero, one of half the values, keys of half their size
                assert bool((bound < want.abs() / 2).float().mean() > 0.99) and d + float(own[3][b, h]) < float(s.min()) / 2


def test_tensors_of_another_place_or_type_are_refused(mx):
    """Host tensors and 64-bit lengths are refused; pinned host memory, which the device reads, is not."""
    g = gen(31)
    cache = make_cache(mx, g, BF16, 2, 40, 16, 2, 64)
    q, lens = rand(g, 2, 4, 64), torch.tensor([40, 7], dtype=torch.int32)
    ws, outs = mx.attn_decode_workspace(cache, 4), []
    for t in (lens.cuda(), lens.pin_memory()):
        outs.append(torch.empty_like(q))
        mx.attn_decode_paged(q, cache, t, 4, 0.125, outs[-1], workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(*outs)
    for bad in (lens, lens.cuda().long()):
        with pytest.raises(mx.MxkError, match="attn_decode_paged"):
            mx.attn_decode_paged(q, cache, bad, 4, 0.125, outs[0], workspace=ws)
    with pytest.raises(mx.MxkError, match="attn_window: .* on cpu"):
        mx.attn_window(q, q.cpu(), q, 2, 2, 4, 4, 64, 0.125, outs[0])


@pytest.mark.parametrize("kind", [BF16, E4M3])
def test_decode_wide_tables_and_short_sequences(mx, kind):
    """Tables with room for far more tokens than there are (the call cannot know), and the same lengths in tables that just
    hold them: other splits of the work, both right."""
    g = gen(25)
    lens = [300, 0, 1, 64, 65, 700]
    cache = make_cache(mx, g, kind, 6, 700, 16, 2, 128)
    wide = torch.full((6, 4000), -1, device="cuda", dtype=torch.int32)
    wide[:, :cache.page_table.shape[1]] = cache.page_table
    for table in (cache.page_table, wide):
        c = mx.KvCache(cache.k, cache.v, table, cache.k_scale, cache.v_scale)
        check_decode(mx, 26, kind, lens, 10, 2, 128, 16, cache=c)
        check_decode(mx, 27, kind, lens, 40, 2, 128, 16, left=90, sinks=3, cache=c)


@pytest.mark.parametrize("kind", [BF16, E4M3])
@pytest.mark.parametrize("D", [48, 64])
@pytest.mark.parametrize("group", [3, 11, 20])
def test_decode_splits_of_short_rows(mx, kind, D, group):
    """Rows of at most 64 channels in every split of the work: tables with room for one to many tiles and few to many sequences,
    lengths at the edges of 64 and 128 tokens and of the pages."""
    g = gen(28)
    edges = [0, 1, 63, 64, 65, 127, 128, 129, 192, 255, 256, 257, 400, 479]
    cache = make_cache(mx, g, kind, len(edges), 480, 16, 2, D)
    for seqs, room, left, sinks in ((3, 100, -1, 0), (14, 256, -1, 0), (14, 300, 140, 5), (14, 4000, -1, 0), (14, 8000, 130, 70), (250, 4000, -1, 0), (250, 500, -1, 0)):
        lens = [min(edges[(5 * i + 3) % len(edges)], room) for i in range(seqs)]
        table = torch.full((seqs, -(-room // 16)), -1, device="cuda", dtype=torch.int32)
        rows = cache.page_table[torch.arange(seqs, device="cuda") % len(edges)][:, :table.shape[1]]
        table[:, :rows.shape[1]] = rows
        c = mx.KvCache(cache.k, cache.v, table, cache.k_scale, cache.v_scale)
        if seqs == 250:  # the plain form for some of them
            q = rand(g, seqs, 2 * group, D)
            out, lse = torch.empty_like(q), torch.empty(seqs, 2 * group, device="cuda")
            sl = torch.tensor(lens, device="cuda", dtype=torch.int32)
            mx.attn_decode_paged(q, c, sl, 2 * group, D ** -0.5, out, lse=lse, workspace=mx.attn_decode_workspace(c, 2 * group))
            few = list(range(0, seqs, 17))
            part = mx.KvCache(cache.k, cache.v, table[few].contiguous(), cache.k_scale, cache.v_scale)
            want = R.decode_reference(q[few], part, [lens[b] for b in few], 2 * group, D ** -0.5, -1, 0)
            R.assert_within(out[few], want[0], want[2], "out")
            R.assert_within(lse[few], want[1], want[3], "lse")
        else:
            check_decode(mx, 29, kind, lens, 2 * group, 2, D, 16, left=left, sinks=sinks, cache=c)


def test_two_streams_at_once(mx):
    """The three calls on two streams at the same time, a workspace each: what they give one after the other."""
    g = gen(60)
    jobs = []
    for i in range(2):
        cache = make_cache(mx, g, BF16, 4, 3000, 16, 2, 128)
        q, qkv = rand(g, 4, 8, 128), rand(g, 2000, 12 * 128)
        jobs.append((cache, q, torch.tensor([3000, 17, 1500 + i, 900], device="cuda", dtype=torch.int32), mx.attn_decode_workspace(cache, 8), qkv))

    def run(job, stream):
        cache, q, lens, ws, qkv = job
        out, big = torch.empty(4, 8, 128, device="cuda", dtype=torch.bfloat16), torch.empty(2000, 8, 128, device="cuda", dtype=torch.bfloat16)
        stream.wait_stream(torch.cuda.current_stream())
        for _ in range(5):
            mx.attn_window(qkv, qkv[:, 1024:], qkv[:, 1280:], 2000, 2000, 8, 2, 128, 0.088, big, left=300, right=0, sinks=4, q_stride=1536, k_stride=1536,
                           v_stride=1536, stream=stream)
            mx.attn_decode_paged(q, cache, lens, 8, 0.088, out, workspace=ws, stream=stream)
        return out, big

    one = [run(j, torch.cuda.default_stream()) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    two = [run(j, s) for j, s in zip(jobs, streams)]
    torch.cuda.synchronize()
    for a, b in zip(one, two):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
