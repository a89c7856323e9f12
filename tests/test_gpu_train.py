"""GPU: the training operators (token order, 8-bit SwiGLU copies, router gradient) against plain implementations in 64 bits.

u = 2^-24 is half a step of fp32, h(type) half a step of the row type (finfo.eps / 2); an output rounded once from fp32 is off by
h |value| plus half the type's smallest step.  The fp32 part of a bound counts the roundings on the way, beside each test."""
import pytest
import torch

import util  # noqa: F401
from util import I

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _check(got, want, fp32_error, what=""):
    """|got - want| within one rounding to the row type plus the fp32 error (a tensor or a number)."""
    got, want = got.cpu(), want.cpu()
    assert got.shape == want.shape
    tiny = torch.finfo(got.dtype).smallest_normal * _half_step(got.dtype) if got.dtype is not torch.float32 else 2.0 ** -149
    bound = _half_step(got.dtype) * (want.abs() + fp32_error) + fp32_error + 2 * tiny
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (what, float((off - bound).max()), float(off.max()))


def oracle_order(idx, El, off=0, align=16, max_rows=None):
    """expert_row0, row_pair, pair_row by a walk over the pairs."""
    T, K = idx.shape
    flat = idx.flatten().tolist()
    lists = [[] for _ in range(El)]
    for i, e in enumerate(flat):
        if 0 <= e - off < El:
            lists[e - off].append(i)
    R = T * K + (align - 1) * El if max_rows is None else max_rows
    row0, row_pair, pair_row, r = [], [-1] * R, [-1] * (T * K), 0
    for pairs in lists:
        row0.append(min(r, R))
        for j, i in enumerate(pairs):
            if r + j < R:
                row_pair[r + j] = i
                pair_row[i] = r + j
        r += -(-len(pairs) // align) * align
    row0.append(min(r, R))
    t = lambda v: torch.tensor(v, dtype=torch.int32)   # noqa: E731
    return t(row0), t(row_pair), t(pair_row).view(T, K)


def _picks(T, K, E, seed, skew=0.0):
    g = _gen(seed)
    logits = torch.randn(T, E, generator=g) + skew * torch.randn(E, generator=g)
    return logits.topk(K, dim=1).indices.to(torch.int32) if T else torch.zeros(0, K, dtype=torch.int32)


def _order(T, K, El, seed, E=None, off=0):
    """(the order on the GPU, its tables on the host)"""
    from justgoal_b200 import TokenOrder
    tables = oracle_order(_picks(T, K, E or El, seed), El, off)
    return TokenOrder(*(t.cuda() for t in tables)), tables


# ------------------------------------------------------------------ sort

@pytest.mark.parametrize("T,K,E,El,off,align", [
    (0, 8, 64, 64, 0, 16), (1, 1, 32, 32, 0, 16), (1, 8, 256, 256, 0, 16), (7, 8, 256, 32, 96, 16), (33, 3, 64, 1, 5, 1), (128, 8, 64, 16, 16, 128),
    (511, 8, 256, 256, 0, 16), (512, 8, 512, 512, 0, 16), (513, 8, 96, 96, 0, 32), (1500, 5, 160, 40, 120, 2), (4097, 1, 32, 32, 0, 64),
    (5000, 8, 512, 512, 0, 8), (14107, 8, 256, 256, 0, 16), (256, 8, 64, 64, 0, 16), (257, 8, 64, 64, 0, 16),
    (160001, 8, 64, 64, 0, 16)])          # (slices of more than one chunk)
def test_sort_tables(T, K, E, El, off, align):
    from justgoal_b200 import sort_tokens
    idx = _picks(T, K, E, seed=T + K, skew=0.7)
    got = sort_tokens(idx.cuda(), El, off, align)
    for g, w, name in zip(got, oracle_order(idx, El, off, align), got._fields):
        assert g.dtype == torch.int32 and torch.equal(g.cpu(), w), name


@pytest.mark.parametrize("T", [64, 700])
def test_sort_strange_ids(T):
    """Ids outside every range, the same expert over and over, everything on one expert, nobody local; ids in a strided view."""
    from justgoal_b200 import sort_tokens
    g = _gen(T)
    wild = torch.randint(-3, 40, (T, 8), generator=g, dtype=torch.int32)
    wild[::5] = torch.tensor([2**31 - 1, -2**31, 7, 7, 7, -1, 33, 0], dtype=torch.int32)
    same = torch.full((T, 8), 9, dtype=torch.int32)
    none = torch.full((T, 8), 100, dtype=torch.int32)
    for idx in (wild, same, none):
        for off in (0, 9):
            for g_, w in zip(sort_tokens(idx.cuda(), 32, off), oracle_order(idx, 32, off)):
                assert torch.equal(g_.cpu(), w)
    wide = torch.cat([wild, wild.flip(0)], dim=1).cuda()
    for g_, w in zip(sort_tokens(wide[:, 8:], 32), oracle_order(wild.flip(0), 32)):
        assert torch.equal(g_.cpu(), w)


@pytest.mark.parametrize("T", [40, 900])
@pytest.mark.parametrize("max_rows", [0, 1, 17, 200])
def test_sort_room_for_fewer_rows(T, max_rows):
    from justgoal_b200 import sort_tokens
    idx = _picks(T, 4, 32, seed=3)
    for g, w in zip(sort_tokens(idx.cuda(), 32, max_rows=max_rows), oracle_order(idx, 32, max_rows=max_rows)):
        assert torch.equal(g.cpu(), w)


# ------------------------------------------------------------------ rows

SIZES = [(1, 1, 32, 128, "bf16"), (5, 8, 32, 128, "fp16"), (37, 3, 64, 384, "fp32"), (200, 8, 32, 1152, "bf16"), (64, 8, 256, 7168, "bf16"),
         (33, 8, 128, 4096, "fp16"), (301, 6, 96, 640, "fp32"), (3000, 2, 32, 256, "bf16"), (0, 8, 32, 256, "bf16"),
         # the combine's gradient by tokens with groups of 32 and 128 threads, by rows with 64, and either side of its line
         (400, 8, 32, 256, "bf16"), (300, 8, 64, 7168, "bf16"), (20, 8, 32, 2048, "bf16"), (256, 7, 32, 512, "fp32"), (257, 7, 32, 512, "fp16")]


def _rows(R, H, dtype, seed, device="cuda"):
    return torch.randn(R, H, generator=_gen(seed)).to(dtype).to(device)


@pytest.mark.parametrize("T,K,E,H,kind", SIZES)
@pytest.mark.parametrize("share", [1, 4])
def test_permute(T, K, E, H, kind, share):
    """Copies: bit for bit; zeros in padding; the rest of the buffer as it was."""
    from justgoal_b200 import permute
    El = E // share
    order, (row0, row_pair, pair_row) = _order(T, K, El, seed=T, E=E, off=0)
    x = _rows(T, H, TYPES[kind], 1)
    out = torch.full((row_pair.numel(), H), 7.0, dtype=TYPES[kind], device="cuda")
    assert permute(x, order, out=out) is out
    used = int(row0[-1])
    want = torch.full((row_pair.numel(), H), 7.0, dtype=TYPES[kind])
    want[:used] = 0
    live = row_pair >= 0
    want[live] = x.cpu()[(row_pair[live] // K).long()]
    assert torch.equal(out.cpu(), want)
    again = permute(x, order)
    assert torch.equal(again[:used].cpu(), want[:used])


@pytest.mark.parametrize("T,K,E,H,kind", SIZES)
def test_restore(T, K, E, H, kind):
    """One product and one rounding: bit for bit the same statement on the host."""
    from justgoal_b200 import quantize_1x128, restore_1x128
    order, (row0, row_pair, pair_row) = _order(T, K, E, seed=T + 1)
    q, scale = quantize_1x128(_rows(T, H, torch.bfloat16, 2))
    flat = (q.cpu().float().view(T, H // 128, 128) * scale.cpu().t()[:, :, None]).view(T, H).to(TYPES[kind])
    assert torch.equal(restore_1x128(q, scale, dtype=TYPES[kind]).cpu(), flat)
    out = torch.full((row_pair.numel(), H), 7.0, dtype=TYPES[kind], device="cuda")
    restore_1x128(q, scale, order, out=out)
    want = torch.full((row_pair.numel(), H), 7.0, dtype=TYPES[kind])
    want[:int(row0[-1])] = 0
    live = row_pair >= 0
    want[live] = flat[(row_pair[live] // K).long()]
    assert torch.equal(out.cpu(), want)


def test_restore_codes_without_a_number_and_signed_zeros():
    from justgoal_b200 import restore_1x128
    q = torch.arange(256, dtype=torch.uint8).view(1, 256).view(torch.float8_e4m3fn).cuda()
    for s in (1.0, 0.37, 2.0 ** -120, 2.0 ** 120, float("nan")):
        scale = torch.full((2, 1), s, device="cuda")
        for dtype in TYPES.values():
            got, want = restore_1x128(q, scale, dtype=dtype).cpu(), (q.cpu().float() * s).to(dtype)
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(torch.signbit(got)[~want.isnan()], torch.signbit(want)[~want.isnan()])
            assert torch.equal(got[~want.isnan()], want[~want.isnan()])


def _combine64(rows, w, tables, T):
    """(sum, sum of magnitudes) per token in 64 bits; rows and w on the host."""
    row0, row_pair, pair_row = tables
    live = (row_pair >= 0).nonzero().flatten()
    pair = row_pair[live].long()
    y = rows[live].double() * w.flatten()[pair].double()[:, None]
    zero = torch.zeros(T, rows.shape[1], dtype=torch.float64)
    token = pair // pair_row.shape[1]
    return zero.index_add(0, token, y), zero.index_add(0, token, y.abs())


@pytest.mark.parametrize("T,K,E,H,kind", SIZES)
@pytest.mark.parametrize("share", [1, 4])
def test_combine_and_permute_backward(T, K, E, H, kind, share):
    """K products and sums by fma: at most K roundings of partial sums, each below the sum of magnitudes."""
    from justgoal_b200 import combine, permute_backward
    order, tables = _order(T, K, E // share, seed=T + 2, E=E)
    rows = _rows(tables[1].numel(), H, TYPES[kind], 3)
    rows[(tables[1] < 0).cuda()] = float("nan")          # nobody may read padding or what lies behind
    w = torch.rand(T, K, generator=_gen(4)) * 2 - 0.5
    for got, weights in ((combine(rows, w.cuda(), order), w), (permute_backward(rows, order), torch.ones(T, K))):
        want, mags = _combine64(rows.cpu(), weights, tables, T)
        assert got.dtype == TYPES[kind]
        _check(got, want, K * U * mags)


@pytest.mark.parametrize("T,K,E,H,kind", SIZES)
@pytest.mark.parametrize("share", [1, 4])
def test_combine_backward(T, K, E, H, kind, share):
    """Rows: one product and one rounding, bit for bit.  Weights: a lane sums at most 8 columns for each of H / 256 steps (32 lanes, the smallest
    CTA), then five shuffles and at most eight partial sums: H / 32 + 13 roundings below the sum of magnitudes."""
    from justgoal_b200 import combine_backward
    order, tables = _order(T, K, E // share, seed=T + 3, E=E)
    row0, row_pair, pair_row = tables
    g, rows = _rows(T, H, TYPES[kind], 5), _rows(row_pair.numel(), H, TYPES[kind], 6)
    rows[(row_pair < 0).cuda()] = float("nan")
    w = torch.rand(T, K, generator=_gen(7)) * 2 - 0.5
    out = torch.full((row_pair.numel(), H), 7.0, dtype=TYPES[kind], device="cuda")
    got, grad_w = combine_backward(g, rows, w.cuda(), order, out=out)
    assert got is out
    want = torch.full((row_pair.numel(), H), 7.0, dtype=TYPES[kind])
    want[:int(row0[-1])] = 0
    live = (row_pair >= 0).nonzero().flatten()
    pair = row_pair[live].long()
    gl = g.cpu()[pair // K]
    want[live] = (gl.float() * w.flatten()[pair][:, None]).to(TYPES[kind])
    assert torch.equal(out.cpu(), want)
    prod = gl.double() * rows.cpu()[live].double()
    dot, mags = torch.zeros(T * K, dtype=torch.float64), torch.zeros(T * K, dtype=torch.float64)
    dot[pair], mags[pair] = prod.sum(dim=1), prod.abs().sum(dim=1)
    assert grad_w.dtype == torch.float32 and grad_w.shape == (T, K)
    _check(grad_w, dot.view(T, K), (H / 32 + 13) * U * mags.view(T, K))


@pytest.mark.parametrize("max_rows", [100, 333])
def test_pairs_without_room_count_as_absent(max_rows):
    """A capacity below the batch's rows: what does not fit has no row, adds nothing and gets no gradient."""
    from justgoal_b200 import combine, combine_backward, permute, permute_backward, sort_tokens
    T, K, H = 60, 6, 256
    idx = _picks(T, K, 32, seed=31)
    tables = oracle_order(idx, 32, max_rows=max_rows)
    order = sort_tokens(idx.cuda(), 32, max_rows=max_rows)
    assert all(torch.equal(a.cpu(), b) for a, b in zip(order, tables)) and bool((tables[2] < 0).any())
    x, g, w = _rows(T, H, torch.float32, 1), _rows(T, H, torch.float32, 2), torch.rand(T, K, generator=_gen(5))
    rows = permute(x, order)
    live = tables[1] >= 0
    assert torch.equal(rows.cpu()[live], x.cpu()[(tables[1][live] // K).long()])
    want, mags = _combine64(rows.cpu(), w, tables, T)
    _check(combine(rows, w.cuda(), order), want, K * U * mags)
    grad_rows, grad_w = combine_backward(g, rows, w.cuda(), order)
    assert bool((grad_w.cpu()[tables[2] < 0] == 0).all()) and bool((grad_w.cpu()[tables[2] >= 0] != 0).all())
    want, mags = _combine64(grad_rows.cpu(), torch.ones(T, K), tables, T)
    _check(permute_backward(grad_rows, order), want, K * U * mags)


def test_order_without_local_pairs_and_without_room():
    from justgoal_b200 import combine, combine_backward, permute, permute_backward, restore_1x128, sort_tokens
    idx = torch.full((9, 4), 50, dtype=torch.int32, device="cuda")
    x, w = _rows(9, 256, torch.bfloat16, 1), torch.ones(9, 4, device="cuda")
    q, scale = torch.ones(9, 256, device="cuda").to(torch.float8_e4m3fn), torch.ones(2, 9, device="cuda")
    for order in (sort_tokens(idx, 16), sort_tokens(idx, 16, 40, max_rows=0)):
        R = order.row_pair.numel()
        assert permute(x, order).shape == (R, 256) and restore_1x128(q, scale, order).shape == (R, 256)
        rows = torch.full((R, 256), float("nan"), dtype=torch.bfloat16, device="cuda")
        assert bool((combine(rows, w, order) == 0).all()) and bool((permute_backward(rows, order) == 0).all())
        grad_rows, grad_w = combine_backward(x, rows, w, order)
        assert grad_rows.shape == (R, 256) and bool((grad_w == 0).all())


def test_tables_of_another_call_stay_inside_the_buffers():
    """Indices outside every range count as -1."""
    from justgoal_b200 import TokenOrder, combine, combine_backward, permute, restore_1x128
    T, K, H, R = 20, 4, 256, 64
    g = _gen(1)
    pair_row = torch.randint(-5, 2 * R, (T, K), generator=g, dtype=torch.int32)
    pair_row[3] = torch.tensor([2**31 - 1, -2**31, R, R - 1], dtype=torch.int32)
    row_pair = torch.randint(-5, 3 * T * K, (R,), generator=g, dtype=torch.int32)
    x, w = _rows(T, H, torch.bfloat16, 1), torch.rand(T, K, generator=g)
    rows = _rows(R, H, torch.bfloat16, 2)
    clean = torch.where((pair_row >= 0) & (pair_row < R), pair_row, -1)
    for last in (0, 10, R, 5 * R, 2**31 - 1):
        row0 = torch.tensor([0, 7, last], dtype=torch.int32)
        wild = TokenOrder(row0.cuda(), row_pair.cuda(), pair_row.cuda())
        tame = TokenOrder(row0.clamp(max=R).cuda(), row_pair.cuda(), clean.cuda())
        big = torch.full((R + 64, H), 3.0, dtype=torch.bfloat16, device="cuda")
        permute(x, wild, out=big[32:32 + R])
        restore_1x128(torch.ones(T, H, device="cuda").to(torch.float8_e4m3fn), torch.ones(H // 128, T, device="cuda"), wild, out=big[32:32 + R])
        combine_backward(x, rows, w.cuda(), wild, out=big[32:32 + R])
        assert bool((big[:32] == 3).all()) and bool((big[32 + R:] == 3).all())
        assert torch.equal(combine(rows, w.cuda(), wild), combine(rows, w.cuda(), tame))


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_views_and_odd_starts_are_copied(kind):
    from justgoal_b200 import combine, combine_backward, permute, permute_backward, swiglu_backward, swiglu_save
    T, K, H = 21, 4, 256
    order, tables = _order(T, K, 32, seed=8)
    R = tables[1].numel()
    dtype = TYPES[kind]

    def odd(t):                       # the same values, one element behind an aligned start
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.flatten()
        return flat[1:].view(t.shape)

    def sliced(t):                    # ... as columns of a wider tensor
        wide = torch.zeros(t.shape[0], t.shape[1] + 40, dtype=t.dtype, device="cuda")
        wide[:, 8:8 + t.shape[1]] = t
        return wide[:, 8:8 + t.shape[1]]

    x, rows, w = _rows(T, H, dtype, 1), _rows(R, H, dtype, 2), torch.rand(T, K, device="cuda")
    used = int(tables[0][-1])
    for form in (odd, sliced, lambda t: t.t().contiguous().t()):
        assert torch.equal(permute(form(x), order)[:used], permute(x, order)[:used])
        assert torch.equal(permute_backward(form(rows), order), permute_backward(rows, order))
        assert torch.equal(combine(form(rows), form(w), order), combine(rows, w, order))
        for a, b in zip(combine_backward(form(x), form(rows), form(w), order), combine_backward(x, rows, w, order)):
            assert torch.equal(a[:used], b[:used])
        saved = swiglu_save(rows)
        for a, b in zip(swiglu_save(form(rows)), saved):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
        d = _rows(R, H // 2, dtype, 3)
        codes = form(saved[1].view(torch.uint8)).view(torch.float8_e4m3fn)
        for a, b in zip(swiglu_backward(codes, form(saved[2]), form(d)), swiglu_backward(saved[1], saved[2], d)):
            assert torch.equal(a, b)


def test_broadcast_gradients():
    """Gradients as a sum's backward pass gives them: one value, expanded."""
    from justgoal_b200 import combine_backward, permute_backward, swiglu_backward, swiglu_save
    order, tables = _order(30, 4, 32, seed=12)
    used, R, H = int(tables[0][-1]), tables[1].numel(), 256
    rows, w, one = _rows(R, H, torch.float32, 1), torch.rand(30, 4, device="cuda"), torch.full((1, 1), 0.5, device="cuda")
    for a, b in zip(combine_backward(one.expand(30, H), rows, w, order), combine_backward(one.repeat(30, H), rows, w, order)):
        assert torch.equal(a[:used], b[:used])
    assert torch.equal(permute_backward(one.expand(R, H), order), permute_backward(one.repeat(R, H), order))
    _, q, scale = swiglu_save(rows)
    for a, b in zip(swiglu_backward(q, scale, one.expand(R, H // 2)), swiglu_backward(q, scale, one.repeat(R, H // 2))):
        assert torch.equal(a, b)


def test_outputs_that_cannot_be_written_are_refused():
    from justgoal_b200 import TokenOrder, combine, combine_backward, permute, restore_1x128, route_backward, swiglu_backward, swiglu_save
    order, tables = _order(8, 4, 32, seed=9)
    R, H = tables[1].numel(), 256
    x, rows, w = _rows(8, H, torch.bfloat16, 1), _rows(R, H, torch.bfloat16, 2), torch.ones(8, 4, device="cuda")
    room = torch.empty(R * H + 8, dtype=torch.bfloat16, device="cuda")
    for out in (room[1:1 + R * H].view(R, H), torch.empty(R, H, device="cuda"), torch.empty(R - 1, H, dtype=torch.bfloat16, device="cuda"),
                torch.empty(H, R, dtype=torch.bfloat16, device="cuda").t(), torch.empty(R, H, dtype=torch.bfloat16)):
        for call in (lambda: permute(x, order, out=out), lambda: combine_backward(x, rows, w, order, out=out)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError, match="share memory"):
        combine_backward(x, rows, w, order, out=rows)
    both = torch.empty(R + 8, H, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        permute(both[:8], order, out=both[4:4 + R])
    with pytest.raises(ValueError, match="share memory"):
        combine(both[:R], w, order, out=both[R - 1:R + 7])
    act, q, scale = swiglu_save(rows)
    with pytest.raises(ValueError, match="share memory"):
        swiglu_save(rows, out=(rows.view(-1)[:R * H // 2].view(R, H // 2), q, scale))
    d = torch.zeros(R, H // 2, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        swiglu_backward(q, scale, d, out=(torch.empty_like(rows), d))
    with pytest.raises(ValueError, match="with_act"):
        swiglu_backward(q, scale, d, with_act=False, out=(torch.empty_like(rows), torch.empty_like(d)))
    with pytest.raises(ValueError):
        restore_1x128(q, scale, order)                                 # another number of tokens
    with pytest.raises(ValueError):
        combine(rows[1:], w, order)
    with pytest.raises(ValueError):
        combine(rows, w.double(), order)
    with pytest.raises(ValueError):
        permute(x[:, :100], order)
    with pytest.raises(ValueError):
        permute(x, TokenOrder(order.expert_row0, order.row_pair.long(), order.pair_row))
    with pytest.raises(ValueError):
        permute(x, TokenOrder(order.expert_row0.cpu(), order.row_pair, order.pair_row))
    logits = torch.zeros(8, 64, device="cuda")
    idx = torch.zeros(8, 4, dtype=torch.int32, device="cuda")
    for bad in (lambda: route_backward(logits[:, :40], None, idx, w, 1.0), lambda: route_backward(logits, None, idx, w, 1.0, 4),
                lambda: route_backward(logits, None, idx, w, 1.0, 6), lambda: route_backward(logits, logits[0], idx, w, 1.0),
                lambda: route_backward(logits, None, idx[:4], w, 1.0), lambda: route_backward(logits, None, idx, w, 1.0, out=logits)):
        with pytest.raises(ValueError):
            bad()


# ------------------------------------------------------------------ SwiGLU and its 8-bit copy

def _copy64(x):
    """Codes (as bytes) and scales of the 8-bit copy, on the host."""
    R, C = x.shape
    g = x.float().view(R, C // 128, 128)
    amax = g.abs().amax(dim=2)
    m, e = torch.frexp(amax.double())
    e = (e - 9 + (m > 0.875).to(e.dtype)).clamp(min=-126)
    scale = torch.ldexp(torch.ones_like(amax, dtype=torch.float64), e)
    scale = torch.where(amax > 0, scale, 1.0)
    scale = torch.where(torch.isfinite(amax), scale, float("nan")).float()
    g = torch.where(scale[:, :, None] == 2.0 ** 120, g.clamp(-240 * 2.0 ** 120, 240 * 2.0 ** 120), g)
    q = (g / scale[:, :, None]).view(R, C).to(torch.float8_e4m3fn)
    return q.view(torch.uint8), scale.t().contiguous()


def _sigmoid_error(gate, dtype):
    """Relative error of the kernel's sigmoid.  16-bit rows: exp within 2 + 1.173 |g| units of 2^-23 (CUDA's bound for the fast
    exponential), the sum half a unit, the fast quotient 2; fp32 rows: exp 2 units, sum and quotient half a unit each."""
    units = 4.5 + 1.173 * gate.abs() if dtype is not torch.float32 else 3.0
    return units * 2 * U


SWIGLU = [(1, 128, "bf16"), (3, 128, "fp32"), (77, 256, "fp16"), (130, 1280, "bf16"), (9, 2048, "bf16"), (1000, 384, "fp16"), (257, 640, "fp32"),
          (5, 8320, "bf16"), (4099, 128, "bf16"), (20003, 256, "bf16")]


@pytest.mark.parametrize("R,inner,kind", SWIGLU)
@pytest.mark.parametrize("part", [1.0, 0.6, 0.0])
def test_swiglu_save(R, inner, kind, part):
    """Codes and scales bit for bit; the activation within the sigmoid's error and two products; rows behind the last as they were."""
    from justgoal_b200 import swiglu_save
    dtype = TYPES[kind]
    used = int(R * part)
    x = torch.randn(R, 2 * inner, generator=_gen(R)) * torch.exp(torch.randn(2 * inner, generator=_gen(R + 1)))
    x[0, :128] = 0.0
    x[R // 2, 5] = -0.0
    x[R // 2, inner:inner + 128] *= 1e-4
    x = x.to(dtype)
    act = torch.full((R, inner), 7.0, dtype=dtype, device="cuda")
    q = torch.full((R, 2 * inner), 9, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.full((2 * inner // 128, R), 7.0, device="cuda")
    row0 = torch.tensor([0, used // 2, used], dtype=torch.int32, device="cuda")
    swiglu_save(x.cuda(), row0, out=(act, q, scale))
    codes, scales = _copy64(x)
    assert torch.equal(q.view(torch.uint8).cpu()[:used], codes[:used]) and torch.equal(scale.cpu()[:, :used], scales[:, :used])
    up, gate = x[:used, :inner].double(), x[:used, inner:].double()
    want = up * gate * torch.sigmoid(gate)
    _check(act[:used], want, want.abs() * (_sigmoid_error(gate, dtype) + 3 * U))
    assert bool((act[used:] == 7).all()) and bool((q.view(torch.uint8)[used:] == 9).all()) and bool((scale[:, used:] == 7).all())
    if used == R:
        for a, b in zip(swiglu_save(x.cuda()), (act, q, scale)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_swiglu_save_scales_at_the_ends(kind):
    """Largest magnitudes around 448 times a power of two, at the ends of the type's range and below 448 * 2^-126."""
    from justgoal_b200 import restore_1x128, swiglu_save
    dtype = TYPES[kind]
    info = torch.finfo(dtype)
    tops = [448.0, 448.0 * (1 + info.eps), 448.0 * (1 - info.eps / 2), 1.75, 1.75 * (1 + info.eps), 224.0, 1.0, info.max, info.smallest_normal,
            info.smallest_normal * info.eps, 448 * 2.0 ** -20]
    if kind != "fp16":
        tops += [448 * 2.0 ** -126, 447 * 2.0 ** -126, 2.0 ** -126, 449 * 2.0 ** -127, 3e38]
    x = torch.rand(len(tops), 256, generator=_gen(2)) * 2 - 1
    x = (x.double() * torch.tensor(tops, dtype=torch.float64)[:, None]).to(dtype)
    x[:, 3] = torch.tensor(tops, dtype=torch.float64).to(dtype)
    x[:, 200] = -torch.tensor(tops, dtype=torch.float64).to(dtype)
    _, q, scale = swiglu_save(x.cuda())
    codes, scales = _copy64(x)
    assert torch.equal(scale.cpu(), scales) and torch.equal(q.view(torch.uint8).cpu(), codes)
    back = restore_1x128(q, scale, dtype=torch.float32).cpu().double()
    step = (scales.double() * 2.0 ** -10).t().repeat_interleave(128, dim=1)          # half of e4m3's smallest step
    assert bool(((back - x.double()).abs() <= torch.maximum(x.double().abs() * 2.0 ** -4, step)).all())


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_swiglu_groups_without_a_number(kind):
    """An infinity or a NaN takes its group of 128 and no other; forward and backward say so."""
    from justgoal_b200 import swiglu_backward, swiglu_save
    dtype = TYPES[kind]
    x = torch.randn(4, 512, generator=_gen(3)).to(dtype)
    x[0, 5], x[1, 130], x[2, 300], x[3, 511] = float("inf"), float("nan"), float("-inf"), float("nan")
    act, q, scale = swiglu_save(x.cuda())
    bad = torch.zeros(4, 4, dtype=torch.bool)
    for r, c in ((0, 0), (1, 1), (2, 2), (3, 3)):
        bad[r, c] = True
    assert torch.equal(scale.isnan().cpu().t(), bad)
    assert bool(q.float().isnan().cpu().view(4, 4, 128)[bad].all()) and not bool(q.float().isnan().cpu().view(4, 4, 128)[~bad].any())
    grad, again = swiglu_backward(q, scale, torch.ones(4, 256, dtype=dtype, device="cuda"))
    touched = (bad[:, :2] | bad[:, 2:])
    g = grad.cpu().view(4, 4, 128)
    assert bool(again.cpu().view(4, 2, 128)[touched].isnan().all()) and bool(torch.isfinite(again.cpu().view(4, 2, 128)[~touched]).all())
    assert bool(g[:, 2:][touched].isnan().all()) and bool(torch.isfinite(g[:, 2:][~touched]).all())
    assert torch.equal(g[:, :2].isnan().all(dim=2), bad[:, 2:]) and torch.equal(g[:, :2].isnan().any(dim=2), bad[:, 2:])


def _grad64(codes, scale, d):
    """(grad of up, of gate, act, |d up|-part of the error terms) in 64 bits from the 8-bit copy."""
    R, C = codes.shape
    x = codes.view(torch.float8_e4m3fn).float().double().view(R, C // 128, 128) * scale.double().t()[:, :, None]
    x = x.view(R, C)
    up, gate, s = x[:, :C // 2], x[:, C // 2:], torch.sigmoid(x[:, C // 2:])
    return up, gate, s, d.double() * gate * s, d.double() * up * s * (1 + gate * torch.sigmoid(-gate)), up * gate * s


@pytest.mark.parametrize("R,inner,kind", SWIGLU)
@pytest.mark.parametrize("part", [1.0, 0.6, 0.0])
def test_swiglu_backward(R, inner, kind, part):
    """d_gate = d up s (1 + gate (1 - s)): the sigmoid's error e counts in s, and |gate| s e + |gate| u (the difference 1 - s) inside the bracket; five
    more roundings."""
    from justgoal_b200 import swiglu_backward
    dtype = TYPES[kind]
    used = int(R * part)
    x = (2 * torch.randn(R, 2 * inner, generator=_gen(R + 5))).to(dtype)
    codes, scale = _copy64(x)
    d = torch.randn(R, inner, generator=_gen(R + 6)).to(dtype)
    grad = torch.full((R, 2 * inner), 7.0, dtype=dtype, device="cuda")
    act = torch.full((R, inner), 7.0, dtype=dtype, device="cuda")
    row0 = torch.tensor([0, used], dtype=torch.int32, device="cuda")
    q = codes.view(torch.float8_e4m3fn).cuda()
    swiglu_backward(q, scale.cuda(), d.cuda(), row0, out=(grad, act))
    up, gate, s, d_up, d_gate, want = (v[:used] for v in _grad64(codes, scale, d))
    e = _sigmoid_error(gate, dtype)
    _check(act[:used], want, want.abs() * (e + 4 * U))
    _check(grad[:used, :inner], d_up, d_up.abs() * (e + 4 * U))
    inside = gate.abs() * (s * e + 2 * U) + U * (1 + gate.abs())
    _check(grad[:used, inner:], d_gate, d_gate.abs() * (e + 5 * U) + (d[:used].double() * up * s).abs() * inside)
    assert bool((act[used:] == 7).all()) and bool((grad[used:] == 7).all())
    alone, none = swiglu_backward(q, scale.cuda(), d.cuda(), with_act=False)
    assert none is None and torch.equal(alone[:used], grad[:used])


def test_swiglu_gates_far_out():
    """Gates at the ends of the range: act = up gate sigma(gate) goes to up gate and to zero, gradients to 1 and 0 times up; nothing becomes NaN."""
    from justgoal_b200 import swiglu_backward, swiglu_save
    gates = torch.tensor([100.0, 3e4, 3e38, -100.0, -3e4, -3.3e38, 0.0, -0.0])
    x = torch.ones(8, 256)
    x[:, 128:] = gates[:, None]
    for dtype in (torch.bfloat16, torch.float32):
        xs = x.to(dtype)
        act, q, scale = swiglu_save(xs.cuda())
        big = xs[:, 128:].double()
        want = torch.where(big > 0, big, torch.zeros_like(big))
        assert bool(torch.isfinite(act).all()) and torch.equal(act.cpu().double(), want)
        grad, again = swiglu_backward(q, scale, torch.ones(8, 128, dtype=dtype, device="cuda"))
        assert not bool(grad.isnan().any()) and not bool(again.isnan().any())
        slope = torch.tensor([1.0, 1, 1, 0, 0, 0, 0.5, 0.5], dtype=torch.float64)[:, None].expand(8, 128)
        assert torch.equal(grad[:, 128:].cpu().double(), slope)


def test_swiglu_gradient_against_differences():
    """Inputs that the 8-bit copy holds exactly (e4m3 values, scale a power of two), moved by h = 2^-4 to either side in fp32: the central
    difference of the kernel's own activation is off by h^2 / 6 |f'''| (|silu'''| < 0.6; up is linear) and by the activations' fp32 errors over h."""
    from justgoal_b200 import swiglu_backward, swiglu_save
    x = torch.randn(16, 512, generator=_gen(11)).clamp(-3, 3).to(torch.float8_e4m3fn).float()
    x[:, ::128] = 3.5                                   # 3.5 = 448 * 2^-7: the scale
    d = torch.ones(16, 256)
    act, q, scale = swiglu_save(x.cuda())
    assert torch.equal(q.float().cpu() * 2.0 ** -7, x)
    grad, again = swiglu_backward(q, scale, d.cuda())
    h = 2.0 ** -4
    for cols, limit in ((slice(0, 256), 0.0), (slice(256, 512), h * h / 6 * 0.6 * 3.5)):
        hi, lo = x.clone(), x.clone()
        hi[:, cols] += h
        lo[:, cols] -= h
        diff = (swiglu_save(hi.cuda())[0].double() - swiglu_save(lo.cuda())[0].double()) / (2 * h)
        off = (diff - grad[:, cols].double()).abs().max()
        assert float(off) <= limit + 2 * 16 * 20 * U / (2 * h), float(off)          # |act| < 16, twenty roundings
    assert torch.equal(again, act)


# ------------------------------------------------------------------ router

MODES = ["deepseek", "renorm_naive", "default", "renormalize", "llama4", "topk"]


def _weights64(mode, logits, bias, idx, factor):
    """The forward's definition in 64 bits, differentiable."""
    at = idx.long()
    x = logits if bias is None or mode == "deepseek" else logits + bias
    if mode == "deepseek":
        s = torch.sigmoid(x).gather(1, at)
        return factor * s / (s.sum(dim=1, keepdim=True) + 1e-20)
    if mode in ("renorm_naive", "renormalize"):
        return factor * torch.softmax(x.gather(1, at), dim=1)
    if mode == "default":
        return factor * torch.softmax(x, dim=1).gather(1, at)
    if mode == "llama4":
        return factor * torch.sigmoid(x.gather(1, at))
    return torch.full(idx.shape, factor / idx.shape[1], dtype=torch.float64) + 0 * logits.sum()


def _route_bound(mode, logits, bias, idx, d, factor):
    """fp32 error of the kernel's formulas: a share or slope is within 16 u (exp 2 units of 2^-23, sum, quotient) plus the rounding of
    the logit's distance to the largest one, 2 u times that distance (and of the biased logit); a sum over the picks adds 8 u; shares and
    sums come up to twice in a product: 64 u + 4 u * span of the terms' magnitudes."""
    x = logits if bias is None or mode == "deepseek" else logits + bias
    at = idx.long()
    span = 2 * x.abs().amax(dim=1, keepdim=True)
    if mode == "deepseek" or mode == "llama4":
        span = 0.0
    rel = 64 * U + 4 * U * span
    if mode == "deepseek":
        s = torch.sigmoid(x).gather(1, at)
        S = s.sum(dim=1, keepdim=True) + 1e-20
        mags = s * torch.sigmoid(-x).gather(1, at) / S * (((d[:, :, None] - d[:, None, :]).abs() * s[:, None, :]).sum(dim=2) + 1e-20 * d.abs()) / S
    elif mode in ("renorm_naive", "renormalize"):
        p = torch.softmax(x.gather(1, at), dim=1)
        mags = p * ((d[:, :, None] - d[:, None, :]).abs() * p[:, None, :]).sum(dim=2)
    elif mode == "default":
        p = torch.softmax(x, dim=1)
        D = torch.zeros_like(p).scatter_add(1, at, d.abs())
        return factor * p * (D * (1 - p) + (p * D).sum(dim=1, keepdim=True)) * rel
    elif mode == "llama4":
        s = x.gather(1, at)
        mags = d.abs() * torch.sigmoid(s) * torch.sigmoid(-s)
    else:
        mags = torch.zeros_like(d)
    return factor * torch.zeros_like(logits).scatter_add(1, at, mags) * rel


def _route_case(mode, T, E, K, seed, spread=1.5, with_bias=True):
    g = _gen(seed)
    logits = spread * torch.randn(T, E, generator=g)
    bias = (0.3 * torch.randn(E, generator=g)).to(torch.bfloat16) if with_bias else None
    idx = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(torch.int32) if T else torch.zeros(0, K, dtype=torch.int32)
    if T:
        idx[::2] = logits[::2].topk(K, dim=1).indices.to(torch.int32)
    return logits, bias, idx, torch.randn(T, K, generator=g)


@pytest.mark.parametrize("mode", MODES)
@pytest.mark.parametrize("T,E,K", [(0, 64, 8), (1, 32, 1), (1, 256, 8), (37, 96, 5), (261, 128, 8), (100, 512, 8), (1025, 256, 2)])
@pytest.mark.parametrize("with_bias", [True, False])
def test_route_backward(mode, T, E, K, with_bias):
    from justgoal_b200 import route_backward
    K = 1 if mode == "llama4" else K
    logits, bias, idx, d = _route_case(mode, T, E, K, seed=T + E + K, with_bias=with_bias)
    got = route_backward(logits.cuda(), None if bias is None else bias.cuda(), idx.cuda(), d.cuda(), 2.5, MODES.index(mode))
    b64 = None if bias is None else bias.double()
    x = logits.double().requires_grad_(True)
    (_weights64(mode, x, b64, idx, 2.5) * d.double()).sum().backward()
    want = x.grad if x.grad is not None else torch.zeros_like(x)
    if mode == "deepseek" and K == 1:             # w = factor s / (s + 1e-20): 64 bits of autograd lose it in the difference
        want = torch.zeros_like(want)
    _check(got, want, _route_bound(mode, logits.double(), b64, idx, d.double(), 2.5) + 1e-18)


@pytest.mark.parametrize("mode", ["deepseek", "renormalize", "default", "llama4"])
def test_route_backward_far_logits(mode):
    """One pick that holds nearly all of the weight, sigmoids near 0 and 1, and sums near the 1e-20 of the definition."""
    from justgoal_b200 import route_backward
    K = 1 if mode == "llama4" else 4
    logits = torch.zeros(6, 64)
    logits[0, 7], logits[1, 7], logits[2], logits[3], logits[4] = 30.0, 12.0, -44.0, -60.0, 40.0
    logits[3, 5], logits[4, 9], logits[5] = -46.0, 80.0, -200.0
    idx = torch.tensor([[7, 9, 5, 3]] * 6, dtype=torch.int32)[:, :K].contiguous()
    d = torch.tensor([[1.0, -2.0, 0.5, 3.0]] * 6)[:, :K].contiguous()
    got = route_backward(logits.cuda(), None, idx.cuda(), d.cuda(), 2.5, MODES.index(mode))
    x, dd, at = logits.double(), d.double(), idx.long()
    p = x.gather(1, at)
    if mode == "deepseek":
        s, slope = torch.sigmoid(p), torch.sigmoid(p) * torch.sigmoid(-p)
        S = s.sum(dim=1, keepdim=True) + 1e-20
        g = slope / S * (((dd[:, :, None] - dd[:, None, :]) * s[:, None, :]).sum(dim=2) + 1e-20 * dd) / S
        want = torch.zeros_like(x).scatter(1, at, 2.5 * g)
    elif mode == "renormalize":
        s = torch.softmax(p, dim=1)
        want = torch.zeros_like(x).scatter(1, at, 2.5 * s * ((dd[:, :, None] - dd[:, None, :]) * s[:, None, :]).sum(dim=2))
    elif mode == "default":
        s = torch.softmax(x, dim=1)
        D = torch.zeros_like(x).scatter(1, at, dd)
        want = 2.5 * s * ((D[:, :, None] - D[:, None, :]) * s[:, None, :]).sum(dim=2)
    else:
        want = torch.zeros_like(x).scatter(1, at, 2.5 * dd * torch.sigmoid(p) * torch.sigmoid(-p))
    # (exp(-200) and exp(-120) are below fp32; 2^-126 is where its full precision ends)
    _check(got, want, _route_bound(mode, x, None, idx, dd, 2.5) + 2.0 ** -126)


@pytest.mark.parametrize("mode", ["deepseek", "renormalize", "default"])
def test_route_backward_strange_ids(mode):
    """An expert named twice gets the sum; ids outside [0, E) carry no weight; a token without picks gets zeros."""
    from justgoal_b200 import route_backward
    logits, bias, idx, d = _route_case(mode, 40, 96, 6, seed=5)
    idx[:, 3] = idx[:, 1]
    idx[::4, 5] = -1
    idx[1::4, 0] = 96
    idx[7] = -1
    got = route_backward(logits.cuda(), bias.cuda(), idx.cuda(), d.cuda(), 1.5, MODES.index(mode))
    x = logits.double().requires_grad_(True)
    total = 0.0
    for t in range(40):
        on = ((idx[t] >= 0) & (idx[t] < 96)).nonzero().flatten()
        if on.numel():
            total = total + (_weights64(mode, x[t:t + 1], bias.double(), idx[t:t + 1, on], 1.5) * d[t:t + 1, on].double()).sum()
    total.backward()
    ok = (idx >= 0) & (idx < 96)
    bound = _route_bound(mode, logits.double(), bias.double(), idx.clamp(0, 95), torch.where(ok, d, 0.0).double(), 1.5).amax(dim=1, keepdim=True)
    _check(got, x.grad, 4 * bound + 1e-18)          # (the bound's own sums count an absent pick's weight as well)
    assert bool((got[7] == 0).all())


@pytest.mark.parametrize("mode", ["deepseek", "renorm_naive", "default", "renormalize", "llama4"])
def test_route_backward_against_differences(mode):
    """Central differences of the layer's own weights: they are fp32 (off by some 16 u of a weight that is at most the factor, over h), and h = 2^-6
    leaves h^2 / 6 times a third derivative below the factor (those of a softmax share or a sigmoid are below 1/4)."""
    import dataclasses
    from justgoal_b200 import MoELayer, route_backward
    shape = {"deepseek": I.TINY_DS, "renorm_naive": I.TINY_RENORM, "default": I.TINY_DEFAULT, "renormalize": I.TINY_RENORMALIZE,
             "llama4": I.TINY_LLAMA4}[mode]
    layer = MoELayer(dataclasses.replace(shape))
    T, E, K, f, h = 4, shape.num_experts, shape.top_k, 2.5, 2.0 ** -6
    g = _gen(21)
    logits = torch.randn(T, E, generator=g)
    boost = torch.randperm(E, generator=g)[:K]
    logits[:, boost] += 4.0                       # picks that a step of h does not change
    if mode == "deepseek":                        # (they lie in at most the groups that are kept)
        logits = torch.randn(T, E, generator=g)
        logits[:, :4] += 4.0
        logits[:, 8:12] += 4.0
    idx, w = layer.route(logits.cuda(), None, f)
    d = torch.randn(T, K, generator=g)
    got = route_backward(logits.cuda(), None, idx, d.cuda(), f, shape.routing_mode).cpu().double()
    for e in sorted(set(idx.flatten().tolist()) | {1, E - 1}):
        loss = []
        for sign in (1, -1):
            moved = logits.clone()
            moved[:, e] += sign * h
            i2, w2 = layer.route(moved.cuda(), None, f)
            assert torch.equal(i2.sort(dim=1).values, idx.sort(dim=1).values)
            by_expert = torch.zeros(T, E, dtype=torch.float64).scatter(1, i2.cpu().long(), w2.cpu().double())
            loss.append((by_expert.gather(1, idx.cpu().long()) * d.double()).sum(dim=1))
        diff = (loss[0] - loss[1]) / (2 * h)
        limit = d.double().abs().sum(dim=1) * f * (h * h / 6 + 16 * U / h)
        assert bool(((diff - got[:, e]).abs() <= limit).all()), (e, (diff - got[:, e]).abs().max(), limit.min())


# ------------------------------------------------------------------ as they are used

class Step:
    """Forward and backward of a layer with fp32 experts through the operators; `keep8`: GEMM1's input rows are made again from an 8-bit copy."""

    def __init__(self, T, E, El, K, H, inner, off, seed, dtype=torch.float32, device="cuda"):
        g = _gen(seed)
        self.shape = I.MoEShape(H, inner, E, El, K, 1, 1, I.ROUTING_RENORMALIZE)
        self.off, self.El, self.K = off, El, K
        mk = lambda *s, scale=1.0: (scale * torch.randn(*s, generator=g)).to(device)   # noqa: E731
        self.x, self.logits, self.grad = mk(T, H).to(torch.bfloat16).to(dtype), mk(T, E), mk(T, H).to(dtype)
        self.w1, self.w2 = mk(El, 2 * inner, H, scale=H ** -0.5).to(dtype), mk(El, H, inner, scale=inner ** -0.5).to(dtype)

    def run(self, layer, keep8):
        import justgoal_b200 as jg
        idx, w = layer.route(self.logits, None, 2.5)
        order = jg.sort_tokens(idx, self.El, self.off)
        row0 = order.expert_row0.tolist()
        seg = [slice(a, b) for a, b in zip(row0, row0[1:])]
        new = lambda c: torch.zeros(order.row_pair.numel(), c, dtype=self.x.dtype, device=self.x.device)   # noqa: E731
        x8 = jg.quantize_1x128(self.x.to(torch.bfloat16)) if keep8 else None
        x_rows = jg.permute(self.x, order, out=new(self.x.shape[1]))
        g_rows, y_rows = new(self.w1.shape[1]), new(self.x.shape[1])
        for e, s in enumerate(seg):
            g_rows[s] = x_rows[s] @ self.w1[e].t()
        act, q, scale = jg.swiglu_save(g_rows, order.expert_row0)
        for e, s in enumerate(seg):
            y_rows[s] = act[s] @ self.w2[e].t()
        out = jg.combine(y_rows, w, order)
        del x_rows, act
        grad_y, grad_w = jg.combine_backward(self.grad, y_rows, w, order)
        grad_act, grad_rows = new(self.w2.shape[2]), new(self.x.shape[1])
        for e, s in enumerate(seg):
            grad_act[s] = grad_y[s] @ self.w2[e]
        grad_g, act = jg.swiglu_backward(q, scale, grad_act, order.expert_row0)
        grad_w1, grad_w2 = torch.zeros_like(self.w1), torch.zeros_like(self.w2)
        x_rows = jg.restore_1x128(*x8, order, dtype=self.x.dtype) if keep8 else jg.permute(self.x, order)
        for e, s in enumerate(seg):
            grad_w2[e] = grad_y[s].t() @ act[s]
            grad_w1[e] = grad_g[s].t() @ x_rows[s]
            grad_rows[s] = grad_g[s] @ self.w1[e]
        grad_x = jg.permute_backward(grad_rows, order)
        grad_logits = jg.route_backward(self.logits, None, idx, grad_w, 2.5, I.ROUTING_RENORMALIZE)
        return {"out": out, "grad_x": grad_x, "grad_w1": grad_w1, "grad_w2": grad_w2, "grad_logits": grad_logits}, idx

    def run64(self, idx, keep8):
        """The same step in 64 bits on the host; the backward pass takes the 8-bit copies where the operators do."""
        x, logits, grad, w1, w2 = (t.double().cpu() for t in (self.x, self.logits, self.grad, self.w1, self.w2))
        idx = idx.cpu().long()
        T, K, inner = x.shape[0], self.K, w2.shape[2]
        p = torch.softmax(logits.gather(1, idx), dim=1)
        out, grad_x, grad_pw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(T, K, dtype=torch.float64)
        gw1, gw2 = torch.zeros_like(w1), torch.zeros_like(w2)
        x8 = x
        if keep8:
            q, s = I.quantize_rows_1x128(self.x.cpu().to(torch.bfloat16))
            x8 = (q.float().view(T, -1, 128) * s.t()[:, :, None]).view(T, -1).double()
        for e in range(self.El):
            t, k = (idx == e + self.off).nonzero(as_tuple=True)
            if not t.numel():
                continue
            w = 2.5 * p[t, k][:, None]
            g = x[t] @ w1[e].t()
            up, gate = g[:, :inner], g[:, inner:]
            y = (up * gate * torch.sigmoid(gate)) @ w2[e].t()
            out.index_add_(0, t, w * y)
            grad_pw[t, k] = (grad[t] * y).sum(dim=1)
            codes, scale = _copy64(g.float())
            up, gate, s, _, _, a = _grad64(codes, scale, torch.zeros(1))
            dy = w * grad[t]
            da = dy @ w2[e]
            dg = torch.cat([da * gate * s, da * up * s * (1 + gate * (1 - s))], dim=1)
            gw2[e], gw1[e] = dy.t() @ a, dg.t() @ x8[t]
            grad_x.index_add_(0, t, dg @ w1[e])
        gl = 2.5 * p * (grad_pw - (p * grad_pw).sum(dim=1, keepdim=True))
        return {"out": out, "grad_x": grad_x, "grad_w1": gw1, "grad_w2": gw2, "grad_logits": torch.zeros_like(logits).scatter(1, idx, gl)}


@pytest.mark.parametrize("T,E,El,off,keep8", [(97, 32, 32, 0, False), (64, 32, 8, 16, True), (1, 32, 32, 0, True)])
def test_a_step_of_training(T, E, El, off, keep8):
    """Route, sort, permute, GEMM1, SwiGLU, GEMM2, combine and all of their gradients, fp32 rows.  Four chains of at most 512 fp32 roundings
    lie behind a gradient, 2048 u = 1.2e-4 of its terms' magnitudes, and terms of random sign add up to some sqrt(512) = 23 times less than those: 2.8e-3 of a
    tensor's norm at worst.  A code of the 8-bit copy that fp32 and 64 bits round to different sides moves a value by 2^-3 of it: one in
    some 2^15 (the products' error of 2^-19 over a step of 2^-4), so 2^-3 / sqrt(2^15) = 7e-4 of a norm."""
    from justgoal_b200 import MoELayer
    step = Step(T, E, El, 4, 256, 128, off, seed=T)
    layer = MoELayer(step.shape)
    got, idx = step.run(layer, keep8)
    want = step.run64(idx, keep8)
    for name, w in want.items():
        off_by = (got[name].double().cpu() - w).norm() / w.norm()
        assert float(off_by) <= 3.5e-3, (name, float(off_by))


def test_wrapped_for_autograd():
    """The pattern of the integration notes: the gradients of the explicit calls, bit for bit."""
    import justgoal_b200 as jg

    class Combine(torch.autograd.Function):
        @staticmethod
        def forward(ctx, rows, topk_w, order):
            ctx.order = order
            ctx.save_for_backward(rows, topk_w)
            return jg.combine(rows, topk_w, order)

        @staticmethod
        def backward(ctx, grad_out):
            return (*jg.combine_backward(grad_out, *ctx.saved_tensors, ctx.order), None)

    order, tables = _order(50, 4, 32, seed=3)
    used = int(tables[0][-1])
    rows, w, g = _rows(tables[1].numel(), 256, torch.float32, 1), torch.rand(50, 4, device="cuda"), _rows(50, 256, torch.float32, 2)
    a, b = rows.clone().requires_grad_(True), w.clone().requires_grad_(True)
    Combine.apply(a, b, order).backward(g)
    grad_rows, grad_w = jg.combine_backward(g, rows, w, order)
    assert torch.equal(a.grad[:used], grad_rows[:used]) and torch.equal(b.grad, grad_w)


def test_streams_graphs_and_repeats():
    """Calls queued on two streams at once, captured and replayed on new inputs, and repeated: the bits of each call made alone."""
    import justgoal_b200 as jg

    def chain(idx, x, w, logits):
        order = jg.sort_tokens(idx, 64)
        rows = jg.permute(x, order, out=torch.zeros(order.row_pair.numel(), x.shape[1], dtype=x.dtype, device="cuda"))
        act, q, scale = jg.swiglu_save(rows, order.expert_row0, out=(torch.zeros(rows.shape[0], 128, dtype=x.dtype, device="cuda"),
                                                                    torch.zeros(rows.shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn),
                                                                    torch.zeros(2, rows.shape[0], device="cuda")))
        back, again = jg.swiglu_backward(q, scale, act, order.expert_row0)
        out = jg.combine(rows, w, order)
        grad, grad_w = jg.combine_backward(out, rows, w, order)
        return (jg.permute_backward(grad, order), grad_w, jg.permute_backward(back, order), order.pair_row, order.expert_row0,
                jg.route_backward(logits, None, idx, grad_w, 1.0), jg.restore_1x128(q, scale, dtype=x.dtype), q.view(torch.uint8), scale)

    def inputs(T, seed):
        g = _gen(seed)
        return (_picks(T, 8, 64, seed).cuda(), torch.randn(T, 256, generator=g).to(torch.bfloat16).cuda(), torch.rand(T, 8, generator=g).cuda(),
                torch.randn(T, 64, generator=g).cuda())

    for T in (5, 1500):
        a, b = inputs(T, 1), inputs(T, 2)
        want_a, want_b = chain(*a), chain(*b)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        got = [[], []]
        for _ in range(5):
            for k, ins in enumerate((a, b)):
                with torch.cuda.stream(streams[k]):
                    got[k].append(chain(*ins))
        torch.cuda.synchronize()
        for k, want in enumerate((want_a, want_b)):
            for res in got[k]:
                for x, y in zip(res, want):
                    assert torch.equal(x, y)
        static = [t.clone() for t in a]
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                res = chain(*static)
            graphs.append((graph, res))
        for ins, want in ((b, want_b), (a, want_a)):
            for s, t in zip(static, ins):
                s.copy_(t)
            for graph, res in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for graph, res in graphs:
                for x, y in zip(res, want):
                    assert torch.equal(x, y)


def test_rows_past_32_bits():
    """A row buffer of more than 2^32 bytes: the last rows are found, written and summed."""
    from justgoal_b200 import TokenOrder, combine, permute
    H, R = 7168, 310000                       # 4.4 GB of bf16
    pair_row = torch.tensor([[0, R - 1], [R - 2, 150001]], dtype=torch.int32, device="cuda")
    row_pair = torch.full((R,), 0, dtype=torch.int32, device="cuda")
    order = TokenOrder(torch.tensor([0, R], dtype=torch.int32, device="cuda"), row_pair, pair_row)
    x = _rows(2, H, torch.bfloat16, 1)
    rows = torch.zeros(R, H, dtype=torch.bfloat16, device="cuda")
    permute(x, order, out=rows)
    assert torch.equal(rows[R - 1], x[0]) and torch.equal(rows[0], x[0]) and torch.equal(rows[R - 2], x[1]) and torch.equal(rows[150001], x[1])
    out = combine(rows, torch.tensor([[1.0, 1.0], [0.5, 0.0]], device="cuda"), order)
    assert torch.equal(out[0], (2 * x[0].float()).to(torch.bfloat16)) and torch.equal(out[1], (0.5 * x[1].float()).to(torch.bfloat16))


def test_swiglu_and_gradients_past_32_bits():
    """More than 2^31 elements in a row buffer: the last rows' activation, 8-bit copy and gradients are those of the same rows alone."""
    from justgoal_b200 import TokenOrder, combine_backward, swiglu_backward, swiglu_save
    R, inner, n = 270000, 4096, 5
    x = torch.zeros(R, 2 * inner, dtype=torch.bfloat16, device="cuda")
    x[-n:] = _rows(n, 2 * inner, torch.bfloat16, 1)
    act, q, scale = swiglu_save(x)
    small = swiglu_save(x[-n:].clone())
    assert torch.equal(act[-n:], small[0]) and torch.equal(q[-n:].view(torch.uint8), small[1].view(torch.uint8)) and torch.equal(scale[:, -n:], small[2])
    assert not bool(act[:7].any()) and bool((scale[:, :7] == 1).all())
    d = torch.zeros(R, inner, dtype=torch.bfloat16, device="cuda")
    d[-n:] = _rows(n, inner, torch.bfloat16, 2)
    grad, again = swiglu_backward(q, scale, d)
    want = swiglu_backward(*small[1:], d[-n:].clone())
    assert torch.equal(grad[-n:], want[0]) and torch.equal(again[-n:], want[1]) and not bool(grad[:7].any())
    del act, q, scale, d, again
    pair_row = torch.tensor([[R - 1, 3]], dtype=torch.int32, device="cuda")
    row_pair = torch.full((R,), -1, dtype=torch.int32, device="cuda")
    row_pair[R - 1], row_pair[3] = 0, 1
    order = TokenOrder(torch.tensor([0, R], dtype=torch.int32, device="cuda"), row_pair, pair_row)
    g, w = _rows(1, 2 * inner, torch.bfloat16, 3), torch.tensor([[0.5, 2.0]], device="cuda")
    grad.fill_(7.0)
    _, grad_w = combine_backward(g, x, w, order, out=grad)
    assert torch.equal(grad[R - 1], (0.5 * g[0].float()).to(torch.bfloat16)) and torch.equal(grad[3], (2 * g[0].float()).to(torch.bfloat16))
    assert not bool(grad[R - 2].any()) and not bool(grad[2].any()) and float(grad_w[0, 1]) == 0.0
    dot = (g[0].double() * x[R - 1].double()).sum()
    assert abs(float(grad_w[0, 0]) - float(dot)) <= (2 * inner / 32 + 13) * U * float((g[0].double() * x[R - 1].double()).abs().sum())


# ------------------------------------------------------------------ orders cut to fewer tokens

@pytest.mark.parametrize("T,all_T", [(20, 40), (400, 500)])          # (the combine's gradient by rows and by tokens)
def test_rows_of_pairs_that_the_call_does_not_have_are_padding(T, all_T):
    """A row in use whose pair is none of the call's T * top_k counts like -1: zeros from every operator that writes rows."""
    from justgoal_b200 import TokenOrder, combine_backward, permute, quantize_1x128, restore_1x128
    K, H = 8, 256
    whole, tables = _order(all_T, K, 32, seed=T)
    order = TokenOrder(whole.expert_row0, whole.row_pair, whole.pair_row[:T])
    row0, row_pair, _ = tables
    used, R = int(row0[-1]), row_pair.numel()
    assert (used > 3 * T and T > 256) == (T == 400)
    here = (row_pair >= 0) & (row_pair < T * K)
    pair = row_pair[here].long()
    x, rows, w = _rows(T, H, torch.bfloat16, 1), _rows(R, H, torch.bfloat16, 2), torch.rand(T, K, generator=_gen(3))
    q, scale = quantize_1x128(x)
    flat = (q.cpu().float().view(T, H // 128, 128) * scale.cpu().t()[:, :, None]).view(T, H).to(torch.bfloat16)
    out = torch.empty(R, H, dtype=torch.bfloat16, device="cuda")
    for name, call, value in (("permute", lambda: permute(x, order, out=out), x.cpu()[pair // K]),
                              ("restore", lambda: restore_1x128(q, scale, order, out=out), flat[pair // K]),
                              ("combine", lambda: combine_backward(x, rows, w.cuda(), order, out=out),
                               (x.cpu()[pair // K].float() * w.flatten()[pair][:, None]).to(torch.bfloat16))):
        out.fill_(float("nan"))
        call()
        want = torch.full((R, H), float("nan"), dtype=torch.bfloat16)
        want[:used] = 0
        want[here] = value
        assert torch.equal(out.cpu().view(torch.int16), want.view(torch.int16)), name


# ------------------------------------------------------------------ outputs that autograd knows

def _calls_with_outputs():
    """(name, the outputs, a call that writes them, the call's inputs) for every operator that takes `out`."""
    import justgoal_b200 as jg
    T, K, H, E = 20, 4, 256, 64
    order, tables = _order(T, K, 32, seed=3)
    R, dtype = tables[1].numel(), torch.bfloat16
    x, rows, w, d = _rows(T, H, dtype, 1), _rows(R, H, dtype, 2), torch.rand(T, K, device="cuda"), _rows(R, H // 2, dtype, 3)
    q8, s8 = jg.quantize_1x128(x)
    _, q, scale = jg.swiglu_save(rows)
    logits, idx = torch.zeros(T, E, device="cuda"), torch.zeros(T, K, dtype=torch.int32, device="cuda")
    new = lambda *shape, dtype=dtype: torch.zeros(*shape, dtype=dtype, device="cuda")   # noqa: E731
    to_rows, to_tokens, to_act, to_q, to_scale = new(R, H), new(T, H), new(R, H // 2), torch.zeros_like(q), torch.zeros_like(scale)
    to_logits = new(T, E, dtype=torch.float32)
    return [("permute", (to_rows,), lambda: jg.permute(x, order, out=to_rows), (x, *order)),
            ("permute_backward", (to_tokens,), lambda: jg.permute_backward(rows, order, out=to_tokens), (rows, *order)),
            ("combine", (to_tokens,), lambda: jg.combine(rows, w, order, out=to_tokens), (rows, w, *order)),
            ("combine_backward", (to_rows,), lambda: jg.combine_backward(x, rows, w, order, out=to_rows), (x, rows, w, *order)),
            ("restore_1x128", (to_rows,), lambda: jg.restore_1x128(q8, s8, order, out=to_rows), (q8, s8, *order)),
            ("swiglu_save", (to_act, to_q, to_scale), lambda: jg.swiglu_save(rows, order.expert_row0, out=(to_act, to_q, to_scale)),
             (rows, order.expert_row0)),
            ("swiglu_backward", (to_rows, to_act), lambda: jg.swiglu_backward(q, scale, d, order.expert_row0, out=(to_rows, to_act)),
             (q, scale, d, order.expert_row0)),
            ("swiglu_backward without act", (to_rows,), lambda: jg.swiglu_backward(q, scale, d, with_act=False, out=(to_rows, None)), (q, scale, d)),
            ("route_backward", (to_logits,), lambda: jg.route_backward(logits, None, idx, w, 1.0, out=to_logits), (logits, idx, w))]


def test_written_outputs_count_as_changed():
    for name, outs, call, ins in _calls_with_outputs():
        before, kept = [t._version for t in outs], [t._version for t in ins]
        call()
        assert all(t._version > v for t, v in zip(outs, before)), name
        assert [t._version for t in ins] == kept, name


def test_a_saved_tensor_that_is_written_again_stops_the_backward_pass():
    """A buffer that a forward pass saved and a later call wrote: the backward pass raises instead of using the new values."""
    import justgoal_b200 as jg
    order, tables = _order(20, 4, 32, seed=4)
    rows, x = _rows(tables[1].numel(), 256, torch.float32, 1), _rows(20, 256, torch.float32, 2)
    weight = torch.ones(256, device="cuda", requires_grad=True)
    loss = (rows * weight).sum()              # saves `rows` for the weight's gradient
    jg.permute(x, order, out=rows)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_a_refused_call_changes_nothing():
    import justgoal_b200 as jg
    rows = _rows(8, 256, torch.bfloat16, 1)
    act, q = torch.zeros(8, 128, dtype=torch.bfloat16, device="cuda"), torch.zeros(8, 256, device="cuda").to(torch.float8_e4m3fn)
    before = act._version, q._version
    with pytest.raises(ValueError):
        jg.swiglu_save(rows, out=(act, q, torch.zeros(3, 8, device="cuda")))
    assert (act._version, q._version) == before


def _forms_with_outputs():
    """name -> (inputs, outputs, call of both lists) for every operator that takes `out`; a call that lets an output lie over an input is refused
    before anything runs."""
    import justgoal_b200 as jg
    T, K, H, E = 20, 4, 256, 64
    order, tables = _order(T, K, 32, seed=3)
    R, bf16, f32 = tables[1].numel(), torch.bfloat16, torch.float32
    new = lambda *shape, dtype=bf16: torch.zeros(*shape, dtype=dtype, device="cuda")   # noqa: E731
    eight = lambda *shape: torch.zeros(*shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)   # noqa: E731
    w, logits, bias, idx = new(T, K, dtype=f32), new(T, E, dtype=f32), new(E), new(T, K, dtype=torch.int32)
    q8, s8, q, scale = eight(T, H), new(H // 128, T, dtype=f32), eight(R, H), new(H // 128, R, dtype=f32)
    t = jg.TokenOrder
    return {
        "permute": ([new(T, H), *order], [new(R, H)], lambda i, o: jg.permute(i[0], t(*i[1:]), out=o[0])),
        "permute_backward": ([new(R, H), order[2]], [new(T, H)], lambda i, o: jg.permute_backward(i[0], t(*order[:2], i[1]), out=o[0])),
        "combine": ([new(R, H), w, order[2]], [new(T, H)], lambda i, o: jg.combine(i[0], i[1], t(*order[:2], i[2]), out=o[0])),
        "combine_backward": ([new(T, H), new(R, H), w, *order], [new(R, H)], lambda i, o: jg.combine_backward(*i[:3], t(*i[3:]), out=o[0])),
        "restore_1x128": ([q8, s8, *order], [new(R, H)], lambda i, o: jg.restore_1x128(*i[:2], t(*i[2:]), out=o[0])),
        "restore_1x128 plain": ([q8, s8], [new(T, H)], lambda i, o: jg.restore_1x128(*i, out=o[0])),
        "swiglu_save": ([new(R, H), order[0]], [new(R, H // 2), eight(R, H), new(H // 128, R, dtype=f32)], lambda i, o: jg.swiglu_save(*i, out=tuple(o))),
        "swiglu_backward": ([q, scale, new(R, H // 2), order[0]], [new(R, H), new(R, H // 2)], lambda i, o: jg.swiglu_backward(*i, out=tuple(o))),
        "route_backward": ([logits, bias, idx, w], [new(T, E, dtype=f32)], lambda i, o: jg.route_backward(*i, 1.0, out=o[0]))}


@pytest.mark.parametrize("name", ["permute", "permute_backward", "combine", "combine_backward", "restore_1x128", "restore_1x128 plain", "swiglu_save",
                                  "swiglu_backward", "route_backward"])
def test_outputs_over_any_input_are_refused(name):
    """Tables, weights, ids and biases as well as rows, and the other outputs: at an output's first bytes and at its last."""
    ins, outs, call = _forms_with_outputs()[name]
    call(ins, outs)                                                     # (apart from each other they are taken)

    def both(a, b, at):                                                 # the two in one buffer, b at byte `at` of a
        room = torch.zeros(at + b.nbytes + a.nbytes, dtype=torch.uint8, device="cuda")
        return room[:a.nbytes].view(a.dtype).view(a.shape), room[at:at + b.nbytes].view(b.dtype).view(b.shape)

    for k, out in enumerate(outs):
        for at in (0, (out.nbytes - 1) // 32 * 32):
            for j, t in enumerate(ins):
                o, i = list(outs), list(ins)
                o[k], i[j] = both(out, t, at)
                with pytest.raises(ValueError, match="share memory"):
                    call(i, o)
            for j in range(k):
                o = list(outs)
                o[k], o[j] = both(out, outs[j], at)
                with pytest.raises(ValueError, match="share memory"):
                    call(ins, o)


def test_sort_in_the_workspace_of_a_larger_batch():
    """One workspace, sized for the largest call, through the C entry point: sizes on both sides of where slices get longer."""
    import ctypes as C
    from justgoal_b200 import _lib
    K, El, most = 8, 64, 37889
    n = C.c_size_t()
    assert _lib.lib.b200moe_sort_workspace_bytes(most, K, El, C.byref(n)) == 0
    room = torch.full((n.value + 64,), 171, dtype=torch.uint8, device="cuda")
    at = room.data_ptr()
    assert at % 16 == 0
    for T in (most, 37888, 300, 20000):
        idx = _picks(T, K, El, seed=T)
        R = T * K + 15 * El
        row0, row_pair, pair_row = (torch.empty(s, dtype=torch.int32, device="cuda") for s in ((El + 1,), (R,), (T, K)))
        ids = idx.cuda()
        rc = _lib.lib.b200moe_sort_tokens(ids.data_ptr(), T, K, El, 0, 16, R, row0.data_ptr(), row_pair.data_ptr(), pair_row.data_ptr(), at, n.value,
                                          torch.cuda.current_stream().cuda_stream)
        assert rc == 0, T
        for g, w in zip((row0, row_pair, pair_row), oracle_order(idx, El)):
            assert torch.equal(g.cpu(), w)
        assert bool((room[n.value:] == 171).all())


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_swiglu_takes_padding_like_any_row(kind):
    """Rows in use are computed whether or not a pair stands in them: zeros give zeros, a NaN stays in its own row, all others as without it."""
    from justgoal_b200 import swiglu_backward, swiglu_save
    dtype = TYPES[kind]
    order, (row0, row_pair, _) = _order(10, 4, 32, seed=6)
    used, R = int(row0[-1]), row_pair.numel()
    padding = (row_pair < 0) & (torch.arange(R) < used)
    first, last = padding.nonzero().flatten()[[0, -1]].tolist()
    x, d = _rows(R, 256, dtype, 1), _rows(R, 128, dtype, 2)
    x[padding.cuda()] = 0
    d[padding.cuda()] = 0
    clean = swiglu_save(x, order.expert_row0)
    grads = swiglu_backward(clean[1], clean[2], d, order.expert_row0)
    on = padding.cuda()
    assert not bool(clean[0][on].any()) and not bool(clean[1][on].float().any()) and bool((clean[2][:, on] == 1).all())
    assert not bool(grads[0][on].any()) and not bool(grads[1][on].any())
    x[first] = float("nan")
    x[last, 200] = float("inf")
    dirty = swiglu_save(x, order.expert_row0)
    grads2 = swiglu_backward(dirty[1], dirty[2], d, order.expert_row0)
    assert bool(dirty[0][first].isnan().all()) and bool(grads2[0][first].isnan().all()) and bool(grads2[1][last].isnan().all())
    rest = torch.arange(used, device="cuda")
    rest = rest[(rest != first) & (rest != last)]
    for a, b in zip((dirty[0], dirty[1].view(torch.uint8), dirty[2].t(), *grads2), (clean[0], clean[1].view(torch.uint8), clean[2].t(), *grads)):
        assert torch.equal(a[rest], b[rest])


@pytest.mark.parametrize("kind", sorted(TYPES))
def test_swiglu_gates_where_the_sigmoid_leaves_the_range(kind):
    """Gates from -84 to -120.  Down to -87 the usual bounds; below, where the sigmoid is under 2^-125, it counts as zero, or has lost bits of its 24
    (fp32 rows, down to -88.7): an output is off by no more than its own size, and never on the other side of zero."""
    from justgoal_b200 import swiglu_backward, swiglu_save
    dtype = TYPES[kind]
    gates = torch.linspace(-84.0, -120.0, 145)
    x = torch.empty(145, 256)
    x[:, :128] = torch.tensor([1.0, -3.0, 0.01, 400.0])[torch.arange(128) % 4]
    x[:, 128:] = gates[:, None]
    x = x.to(dtype)

    def check(got, want, gate, usual):
        _check(got, want, torch.where(gate < -87, want.abs(), usual))
        assert bool((got.cpu().double() * want >= 0).all())

    act, q, scale = swiglu_save(x.cuda())
    up, gate = x[:, :128].double(), x[:, 128:].double()
    want = up * gate * torch.sigmoid(gate)
    check(act, want, gate, want.abs() * (_sigmoid_error(gate, dtype) + 3 * U))
    d = torch.tensor([1.0, -0.5])[torch.arange(128) % 2].repeat(145, 1).to(dtype)
    grad, again = swiglu_backward(q, scale, d.cuda())
    up, gate, s, d_up, d_gate, want = _grad64(*_copy64(x), d)
    e = _sigmoid_error(gate, dtype)
    check(again, want, gate, want.abs() * (e + 4 * U))
    check(grad[:, :128], d_up, gate, d_up.abs() * (e + 4 * U))
    check(grad[:, 128:], d_gate, gate, d_gate.abs() * (e + 5 * U) + (d.double() * up * s).abs() * (gate.abs() * (s * e + 2 * U) + U * (1 + gate.abs())))


# ------------------------------------------------------------------ loops of large calls

@pytest.mark.parametrize("T,K,E,H,kind", [
    # by tokens, more tokens than the grid takes in one turn (2368 CTAs of four tokens, of two, of one), rows of 128 columns among them
    (9601, 4, 32, 128, "bf16"), (9601, 5, 64, 128, "fp32"), (9602, 4, 32, 128, "fp16"), (400, 8, 32, 128, "bf16"), (300, 6, 64, 128, "fp32"), (9601, 4, 64, 256, "fp16"),
    (5001, 6, 64, 1152, "bf16"), (4999, 4, 32, 640, "fp32"), (2501, 5, 96, 2176, "bf16"), (2500, 4, 32, 1152, "fp32"), (4750, 8, 256, 384, "bf16"),
    # by rows, several turns of groups of 32, 64 and 128 threads
    (256, 8, 256, 128, "bf16"), (64, 8, 256, 2048, "bf16"), (64, 8, 256, 2048, "fp32"), (16, 8, 512, 7168, "fp16"), (9601, 2, 32, 128, "bf16")])
def test_combine_backward_many_turns(T, K, E, H, kind):
    test_combine_backward(T, K, E, H, kind, 1)


@pytest.mark.parametrize("op", ["permute", "restore", "combine_backward"])
def test_padding_behind_a_warps_first_block(op):
    """More rows than 32 per warp of the grid: zeros in those without a pair, the rest as it was."""
    from justgoal_b200 import TokenOrder, combine_backward, permute, restore_1x128
    T, R, H = (300, 300001, 128) if op == "combine_backward" else (1, 300001, 128)
    row_pair = torch.zeros(R, dtype=torch.int32)
    row_pair[::3] = -1
    row_pair[-40:] = -1
    row_pair[1::7] = 2 * T                                   # a pair of another call
    used = R - 5
    pair_row = torch.full((T, 1), -1, dtype=torch.int32)
    pair_row[0] = 250004
    row_pair[250004] = 0
    order = TokenOrder(torch.tensor([0, used], dtype=torch.int32, device="cuda"), row_pair.cuda(), pair_row.cuda())
    x = _rows(T, H, torch.bfloat16, 1)
    out = torch.full((R, H), 7.0, dtype=torch.bfloat16, device="cuda")
    if op == "permute":
        permute(x, order, out=out)
    elif op == "restore":
        restore_1x128(x.to(torch.float8_e4m3fn), torch.ones(1, T, device="cuda"), order, out=out)
        x = x.to(torch.float8_e4m3fn).to(torch.bfloat16)
    else:
        combine_backward(x, torch.zeros(R, H, dtype=torch.bfloat16, device="cuda"), torch.ones(T, 1, device="cuda"), order, out=out)
    want = torch.full((R, H), 7.0, dtype=torch.bfloat16)
    want[:used][(row_pair[:used] < 0) | (row_pair[:used] >= T)] = 0
    want[250004] = x[0].cpu()
    assert torch.equal(out.cpu(), want)


# (rows per CTA and groups per row of the walks: several turns, and rows that end inside a block)
BLOCKS = [(3001, 640, "bf16"), (2499, 640, "fp32"), (5003, 384, "fp16"), (5003, 384, "fp32"), (1001, 1664, "bf16"), (601, 8320, "bf16"), (9501, 128, "fp32")]


@pytest.mark.parametrize("R,inner,kind", BLOCKS)
@pytest.mark.parametrize("part", [1.0, 0.87])
def test_swiglu_save_of_several_turns(R, inner, kind, part):
    """As test_swiglu_save.  Gates below -87, which the larger draws hold: the sigmoid counts as zero there (or, in fp32 rows down to -88.7, loses bits of
    its 24 below the normal range), so the activation, e^-87 of up gate at most, is off by no more than itself."""
    from justgoal_b200 import swiglu_save
    dtype, used = TYPES[kind], int(R * part)
    x = torch.randn(R, 2 * inner, generator=_gen(R)) * torch.exp(torch.randn(2 * inner, generator=_gen(R + 1)))
    x[0, :128] = 0.0
    x[R // 2, 5] = -0.0
    x[R // 2, inner:inner + 128] *= 1e-4
    x = x.to(dtype)
    act = torch.full((R, inner), 7.0, dtype=dtype, device="cuda")
    q = torch.full((R, 2 * inner), 9, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale = torch.full((2 * inner // 128, R), 7.0, device="cuda")
    swiglu_save(x.cuda(), torch.tensor([0, used], dtype=torch.int32, device="cuda"), out=(act, q, scale))
    codes, scales = _copy64(x)
    assert torch.equal(q.view(torch.uint8).cpu()[:used], codes[:used]) and torch.equal(scale.cpu()[:, :used], scales[:, :used])
    up, gate = x[:used, :inner].double(), x[:used, inner:].double()
    want = up * gate * torch.sigmoid(gate)
    _check(act[:used], want, want.abs() * torch.where(gate < -87, 1.0, _sigmoid_error(gate, dtype) + 3 * U))
    assert bool((act[used:] == 7).all()) and bool((q.view(torch.uint8)[used:] == 9).all()) and bool((scale[:, used:] == 7).all())


@pytest.mark.parametrize("R,inner,kind", BLOCKS)
@pytest.mark.parametrize("part", [1.0, 0.87])
def test_swiglu_backward_of_several_turns(R, inner, kind, part):
    test_swiglu_backward(R, inner, kind, part)


@pytest.mark.parametrize("T,K,E,El,off,align", [(160001, 8, 512, 512, 0, 16), (170003, 8, 256, 200, 40, 32), (310001, 8, 512, 509, 2, 1)])
def test_sort_slices_of_several_chunks(T, K, E, El, off, align):
    test_sort_tables(T, K, E, El, off, align)


@pytest.mark.parametrize("T,K,E,H,kind", [(253, 3, 32, 7168, "bf16"), (254, 3, 32, 7168, "bf16"), (888, 2, 32, 2048, "fp16"), (889, 2, 32, 2048, "fp16"), (444, 8, 64, 2048, "fp32"),
                                          (445, 8, 64, 2048, "fp32"), (100, 8, 256, 1920, "bf16"), (9000, 1, 32, 128, "fp32")])
def test_rows_on_both_sides_of_the_ctas_sizes(T, K, E, H, kind):
    """CTAs of 64 and of 128 threads (and of 256, for rows read back without an order)."""
    test_permute(T, K, E, H, kind, 1)
    test_permute(T, K, E, H, kind, 4)
    test_restore(T, K, E, H, kind)


@pytest.mark.parametrize("R,inner,kind", [(77, 4096, "bf16"), (3, 8320, "fp32"), (200, 4224, "fp16"), (591, 2048, "bf16"), (592, 2048, "fp32"), (1183, 1536, "bf16"),
                                          (1186, 640, "fp32"), (2400, 640, "bf16"), (2367, 384, "fp16")])
def test_swiglu_blocks_of_few_rows(R, inner, kind):
    """Blocks that are halved, in rows or in groups, until there are four CTAs per SM, and those on the line."""
    test_swiglu_save_of_several_turns(R, inner, kind, 1.0)
    test_swiglu_save_of_several_turns(R, inner, kind, 0.87)
    test_swiglu_backward(R, inner, kind, 0.87)


def test_fp16_rows_at_the_end_of_their_range():
    """65504 has the code of 65536: finite in fp32 and bf16, an infinity where it is restored as fp16; the gradients, made in fp32, are finite."""
    from justgoal_b200 import restore_1x128, swiglu_backward, swiglu_save
    x = torch.full((2, 256), 65504.0, dtype=torch.float16)
    x[:, 128:] = 0.5
    x[1, :128] = -63488.0                                # (half-way, to the even code: 256)
    x[1, 1:128] = -63456.0                               # ... and the next smaller: 240
    _, q, scale = swiglu_save(x.cuda())
    for dtype in (torch.float32, torch.bfloat16):
        back = restore_1x128(q, scale, dtype=dtype)
        assert bool((back[0, :128] == 65536).all()) and float(back[1, 0]) == -65536 and bool((back[1, 1:128] == -61440).all())
    assert bool(restore_1x128(q, scale, dtype=torch.float16)[0, :128].isinf().all())
    grad, act = swiglu_backward(q, scale, torch.full((2, 128), 1e-3, dtype=torch.float16, device="cuda"))
    assert bool(torch.isfinite(grad).all()) and bool(torch.isfinite(act).all())
