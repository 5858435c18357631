"""GPU tests of the paged 8-bit cache's operators (paged_plan, paged_append,
paged_attention) against plain 64-bit implementations (paged_ref.py)."""
import math
import random

import pytest
import torch

import paged_ref as ref
import pmkl_b200
import pmkl_pytorch_ext
from pmkl_function import paged_append, paged_attention, paged_plan

pytestmark = pytest.mark.gpu

KERNELS = [0, 1, 2, 3]  # PMKL_PAGED_AUTO, _SIMT, _STREAM, _TCGEN05
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_timeouts():
    yield
    assert pmkl_b200.device_error(clear=True) == 0, "a kernel abandoned a bounded wait"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ---------------------------------------------------------------- plan
def run_plan(cached, new, table, free, count, block, max_tokens):
    t = i32(table).reshape(len(cached), -1)
    free_d = i32(free + [-7])  # a capacity past the count
    seq, starts, slots, left, status = paged_plan(i32(cached), i32(new), t, free_d, i32([count]), block, max_tokens)
    want = ref.plan(cached, new, table, free, count, block, max_tokens)
    got = (seq.tolist(), starts.tolist(), slots.tolist(), left.item(), status.tolist(), t.tolist())
    assert got[0] == want[0] and got[1] == want[1] and got[3] == want[3] and got[4] == want[4]
    assert got[2] == want[2]
    assert got[5] == [list(r) for r in want[5]]
    return want


def random_plan(seed, batch, block, max_len, max_new, spare, pad, width_cut=0):
    r = random.Random(seed)
    cached = [r.randint(0, max_len) for _ in range(batch)]
    new = [r.randint(0, max_new) for _ in range(batch)]
    width = max(1, max(-(-(c + n) // block) for c, n in zip(cached, new)) - width_cut)
    held = sum(-(-c // block) for c in cached)
    need = sum(-(-(c + n) // block) - -(-c // block) for c, n in zip(cached, new))
    pool = list(range(held + max(0, need + spare)))
    r.shuffle(pool)
    table, at = [], 0
    for c in cached:
        k = min(width, -(-c // block))
        table.append(pool[at:at + k] + [-1] * (width - k))
        at += k
    free = pool[held:]
    return cached, new, table, free, len(free), block, max(0, sum(new) + pad)


@pytest.mark.parametrize("batch", [1, 2, 31, 255, 256, 257, 700])
@pytest.mark.parametrize("block,max_len,max_new", [(16, 100, 1), (1, 9, 5), (7, 50, 40), (128, 1000, 300)])
def test_plan_random(batch, block, max_len, max_new):
    want = run_plan(*random_plan(batch * 1000 + block, batch, block, max_len, max_new, spare=3, pad=5))
    assert not any(want[4])


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("spare,pad,cut", [(-7, 0, 0), (0, -60, 0), (2, 0, 2), (-9, -40, 1), (-10 ** 6, 3, 0)])
def test_plan_leaves_requests_out(seed, spare, pad, cut):
    """Too few pages, tokens or columns: the same requests as the definition's are left out."""
    want = run_plan(*random_plan(seed, 300, 8, 60, 25, spare=spare, pad=pad, width_cut=cut))
    assert any(want[4])


def test_plan_long_prompts_and_empty():
    run_plan([0, 33], [65537, 0], [[-1] * 4100, [3, 9, 4] + [-1] * 4097], list(range(10, 5000)), 4990, 16, 65537 + 9)
    run_plan([5, 0], [0, 0], [[1], [-1]], [], 0, 16, 0)
    run_plan([-3], [-2], [[-1]], [4], 1, 16, 3)  # negative lengths count as 0
    seq, starts, slots, left, status = paged_plan(i32([]), i32([]), i32([]).reshape(0, 4), i32([1, 2]), i32([2]), 16, 4)
    assert starts.tolist() == [0] and slots.tolist() == [-1] * 4 and left.item() == 2 and seq.numel() == 0


def test_plan_lengths_past_31_bits():
    """A request whose length would not fit in 32 bits is left out, and the next one is not."""
    top = 2 ** 31 - 1
    seq, starts, slots, left, status = paged_plan(i32([top - 1, top - 1]), i32([4, 1]), i32([[5, 6, -1], [7, 8, -1]]), i32([9]),
                                                  i32([1]), 1 << 30, 6)
    assert status.tolist() == [2, 0] and seq.tolist() == [top - 1, top]
    assert starts.tolist() == [0, 4, 5] and left.item() == 1
    assert slots.tolist() == [-1] * 4 + [8 * (1 << 30) + (top - 1 - (1 << 30)), -1]


# ---------------------------------------------------------------- append
def run_append(xk, xv, slots, kc, vc, ks, vs):
    """paged_append on CUDA copies; caches bit for bit as the definition says."""
    dev = [t.cuda() for t in (kc, vc, ks, vs)]
    paged_append(xk, xv, torch.tensor(slots, dtype=torch.int64, device="cuda"), *dev)
    for x, c0, s0, c1, s1 in ((xk, kc, ks, dev[0], dev[2]), (xv, vc, vs, dev[1], dev[3])):
        want, scale = ref.append(x.cpu(), slots, c0, s0)
        assert torch.equal(s1.cpu().double(), scale)
        got = c1.cpu().double()
        assert torch.equal(torch.nan_to_num(got, nan=1e4), torch.nan_to_num(want, nan=1e4))
    return dev


def values(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[:-1] + (1,), generator=g))
    return x.to(dtype).cuda()


def run_slots(runs, block):
    """Slots of runs (page, first row, rows); page None: a token without a slot."""
    out = []
    for page, row, n in runs:
        out += [-1] * n if page is None else [page * block + row + i for i in range(n)]
    return out


@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("heads,hidden,block", [(1, 64, 16), (3, 128, 16), (2, 128, 64), (2, 80, 16), (5, 7, 3), (1, 256, 1),
                                                (2, 64, 128), (4, 24, 33)])
@pytest.mark.parametrize("rows_first", [False, True])
def test_append_runs(dtype, heads, hidden, block, rows_first):
    b = block
    runs = [(4, 0, b), (2, b - 1, 1), (1, 0, max(1, b // 2)), (None, 0, 2), (7, b // 2, b - b // 2), (0, 0, b), (3, 0, 1), (6, b // 3, 1)]
    slots = run_slots(runs, b)
    caches = [ref.make_cache(8, heads, b, hidden, seed=s, rows_first=rows_first) for s in (1, 2)]
    xk, xv = (values((len(slots), heads, hidden), dtype, s) for s in (3, 4))
    run_append(xk, xv, slots, caches[0][0], caches[1][0], caches[0][1], caches[1][1])


def test_append_token_by_token_equals_any_split():
    """A page filled token by token: scales are those of the whole page, values at most re-rounded."""
    heads, hidden, block = 2, 64, 16
    x = values((block, heads, hidden), BF16, 5, spread=2.0)
    kc, ks = ref.make_cache(3, heads, block, hidden, seed=6)
    whole = run_append(x, x, run_slots([(1, 0, block)], block), kc, kc, ks, ks)
    step = [t.cuda() for t in (kc, kc, ks, ks)]
    for i in range(block):
        one = [t.cpu() for t in step]
        step = run_append(x[i:i + 1], x[i:i + 1], [block + i], one[0], one[1], one[2], one[3])
    assert torch.equal(step[2], whole[2])
    a, b = step[0][1].float(), whole[0][1].float()
    assert ((a - b).abs() <= 2.0 ** -9 * block).all()  # subnormals only


def test_append_special_values():
    heads, hidden, block = 2, 64, 16
    x = values((6, heads, hidden), BF16, 7).float()
    x[0, 0, 3], x[1, 0, 5], x[2, 1, :] = math.nan, math.inf, 0.0
    x[3, 1, 9] = -math.inf
    x[4] = 0.0
    x[5, 0, 0] = 3e38
    slots = run_slots([(0, 0, 2), (1, 3, 1), (2, 0, 1), (3, 0, 1), (4, 2, 1)], block)
    kc, ks = ref.make_cache(5, heads, block, hidden, seed=8)
    run_append(x.cuda(), (x * 1e-30).cuda(), slots, kc, kc, ks, ks)
    # powers of two and 448 times them: the scale's edges
    e = torch.tensor([448.0, 449.0, 447.9, 1.75, 1.7500001, 0.875, 2.0 ** -60, 2.0 ** -80])
    y = torch.zeros(8, 1, 8)
    y[:, 0, 2] = -e
    kc, ks = ref.make_cache(8, 1, 4, 8, seed=9)
    run_append(y.cuda(), y.cuda(), [4 * i for i in range(8)], kc, kc, ks, ks)


def test_append_strided_inputs_and_foreign_slots():
    heads, hidden, block = 3, 64, 16
    big = values((9, 2 * heads + 1, hidden), F16, 10)
    kc, ks = ref.make_cache(2, heads, block, hidden, seed=11)
    slots = [0, 1, 2, -1, 2 * block, 1 << 40, 17, 18, -5]  # outside the cache: skipped
    run_append(big[:, :heads], big[:, heads:2 * heads], slots, kc, kc, ks, ks)


# ---------------------------------------------------------------- attention
def problem(lens, news, H, Hkv, D, block, dtype, seed, rows_first=False, poison=True, width_extra=1, tail=0, std=1.0):
    """A cache whose unused rows, pages and table entries are poisoned."""
    pages = sum(-(-n // block) for n in lens) + 2
    kc, ks = ref.make_cache(pages, Hkv, block, D, seed, rows_first)
    vc, vs = ref.make_cache(pages, Hkv, block, D, seed + 1, rows_first)
    r = random.Random(seed)
    pool = list(range(pages))
    r.shuffle(pool)
    width = max([1] + [-(-n // block) for n in lens]) + width_extra
    table, used = [], torch.zeros(pages, block, dtype=torch.bool)
    for n in lens:
        k = -(-n // block)
        row = [pool.pop() for _ in range(k)]
        for j, p in enumerate(row):
            used[p, :min(block, n - j * block)] = True
        table.append(row + [r.choice([-1, 1 << 30, 0])] * (width - k))
    if poison:
        for c in (kc, vc):
            c.view(torch.uint8)[~used[:, None, :].expand(pages, Hkv, block)] = 0x7F  # NaN
        for s in (ks, vs):
            s[~used.any(1)] = math.nan
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    g = torch.Generator().manual_seed(seed + 2)
    q = (torch.randn(starts[-1] + tail, H, D, generator=g) * std).to(dtype)
    return q, kc, vc, ks, vs, table, lens, starts


def needs(kernel, dtype, D=64, block=16):
    """Skips what a kernel asked for by name does not cover."""
    if kernel >= 2 and (D not in (64, 128) or block % 16):
        pytest.skip("not this kernel's head or page size")
    if kernel == 3 and dtype == F32:
        pytest.skip("16-bit queries only")


def check(prob, causal=True, scale=0.0, kernel=0, with_starts=True, q_dev=None):
    needs(kernel, prob[0].dtype, prob[0].shape[2], prob[1].shape[2])
    q, kc, vc, ks, vs, table, lens, starts = prob
    want, lse, weight = ref.attention(q, kc, vc, ks, vs, table, lens, starts, causal, scale)
    news = [b - a for a, b in zip(starts, starts[1:])]
    out, got_lse = pmkl_pytorch_ext.paged_attention_fw(
        q.cuda() if q_dev is None else q_dev, kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), i32(table), i32(lens),
        i32(starts) if with_starts else None, max(news), causal, scale, kernel)
    o = out.cpu().double()
    assert out.dtype == q.dtype and o.isfinite().all()
    bound = ref.out_bound(want, weight, lse, q.dtype, max(lens + [1]))
    err = (o - want).abs()
    assert (err <= bound).all(), f"out: err {err.max():.3e}, worst err / bound {(err / bound).max():.3f}"
    empty = lse.isinf()
    l = got_lse.cpu().double()
    assert torch.equal(l.isinf(), empty) and (l[empty] < 0).all() and (o[empty] == 0).all()
    assert ((l - lse).abs()[~empty] <= ref.lse_bound(lse)[~empty]).all()
    return out, got_lse


LENS = [1, 15, 16, 17, 31, 127, 128, 129, 300, 0, 513]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,D,block", [(4, 4, 64, 16), (8, 2, 128, 16), (6, 1, 128, 64), (8, 1, 64, 128), (3, 3, 128, 32),
                                           (4, 2, 96, 16), (2, 1, 64, 7), (2, 2, 256, 16), (5, 5, 33, 1), (10, 1, 128, 48)])
def test_attention_one_token(kernel, dtype, H, Hkv, D, block):
    """One query a request, lengths from 0 to a few pages, unused rows NaN, unused entries out of range."""
    check(problem(LENS, [1] * len(LENS), H, Hkv, D, block, dtype, seed=D + block), kernel=kernel, with_starts=block != 16)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,D,block", [(4, 4, 64, 16), (8, 2, 128, 32), (8, 1, 128, 16), (3, 1, 64, 128), (4, 2, 40, 5)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_several_tokens(kernel, dtype, H, Hkv, D, block, causal):
    """Several queries a request (0 to 70), among them requests with more queries than keys: rows without a key."""
    lens, news = [64, 1, 200, 7, 130, 90, 0, 33], [3, 1, 5, 9, 0, 70, 2, 33]
    check(problem(lens, news, H, Hkv, D, block, dtype, seed=block + D, rows_first=True, tail=3), causal=causal, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_long(kernel, dtype):
    """Lengths that many CTAs share."""
    check(problem([5000, 3, 2111], [1, 1, 1], 4, 2, 128, 16, dtype, seed=1), kernel=kernel)
    check(problem([4097], [2], 8, 1, 64, 64, dtype, seed=2), kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_attention_peaked_and_scaled(kernel, dtype):
    """Scores that grow along the keys and pages of very different scales."""
    prob = problem([700, 257], [1, 2], 4, 2, 128, 16, dtype, seed=3, std=2.0)
    ks, vs = prob[3], prob[4]
    ks *= torch.exp2(torch.arange(ks.shape[0])[:, None] % 5 - 2.0)
    vs *= torch.exp2(torch.arange(vs.shape[0])[:, None] % 31 - 15.0)
    check(prob, kernel=kernel)
    check(prob, scale=0.01, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_missing_pages(kernel):
    """Keys in pages outside the cache count as not there; a request of such pages only gives empty rows."""
    prob = problem([100, 48, 80], [1, 1, 4], 4, 2, 64, 16, F16, seed=4)
    table = prob[5]
    table[0][2], table[0][6] = -1, 1 << 20
    table[1][0], table[1][1], table[1][2] = -5, -1, 10 ** 9
    check(prob, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_strided_queries(kernel):
    prob = list(problem([33, 129], [1, 3], 4, 2, 64, 16, BF16, seed=5))
    wide = torch.zeros(4, 4, 3, 64, dtype=BF16, device="cuda")
    view = wide[:, :, 1]
    view.copy_(prob[0])
    assert not view.is_contiguous()
    check(prob, kernel=kernel, q_dev=view)
    odd = torch.zeros(4 * 4 * 64 + 3, dtype=BF16, device="cuda")[3:].view(4, 4, 64)  # a base of 2-byte alignment
    odd.copy_(prob[0])
    check(prob, kernel=kernel, q_dev=odd)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_nan_and_inf_queries_stay_in_their_rows(kernel, dtype):
    needs(kernel, dtype)
    q, kc, vc, ks, vs, table, lens, starts = problem([200, 90], [2, 1], 8, 2, 128, 16, dtype, seed=6)
    args = [t.cuda() for t in (kc, vc, ks, vs)] + [i32(table), i32(lens), i32(starts), 2, True, 0.0, kernel]
    clean, clean_lse = pmkl_pytorch_ext.paged_attention_fw(q.cuda(), *args)
    bad = q.clone()
    bad[0, 1, 5], bad[1, 6, 0] = math.nan, math.inf
    out, lse = pmkl_pytorch_ext.paged_attention_fw(bad.cuda(), *args)
    assert out[0, 1].isnan().all() and out[1, 6].isnan().any()
    keep = torch.ones(q.shape[:2], dtype=torch.bool)
    keep[0, 1] = keep[1, 6] = False
    assert torch.equal(out[keep.cuda()], clean[keep.cuda()]) and torch.equal(lse[keep.cuda()], clean_lse[keep.cuda()])


@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_same_bits_again_and_on_another_stream(kernel):
    q, kc, vc, ks, vs, table, lens, starts = problem([900, 31, 4000], [1, 4, 1], 8, 2, 128, 16, BF16, seed=7)
    args = [t.cuda() for t in (q, kc, vc, ks, vs)] + [i32(table), i32(lens), i32(starts), 4, True, 0.0, kernel]
    a = pmkl_pytorch_ext.paged_attention_fw(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        b = pmkl_pytorch_ext.paged_attention_fw(*args)
    side.synchronize()
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_step_in_a_graph():
    """plan, append and attention captured once and replayed with other lengths and values."""
    H, Hkv, D, block, B, width = 4, 2, 64, 16, 3, 8
    cached, new = i32([0, 0, 0]), i32([0, 0, 0])
    table = torch.full((B, width), -1, dtype=torch.int32, device="cuda")
    free, count = torch.arange(24, dtype=torch.int32, device="cuda"), i32([24])
    kc, vc = (torch.zeros(24, Hkv, block, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = torch.ones(24, Hkv, device="cuda"), torch.ones(24, Hkv, device="cuda")
    k, v = (torch.zeros(12, Hkv, D, device="cuda", dtype=BF16) for _ in range(2))
    q = torch.zeros(12, H, D, device="cuda", dtype=BF16)

    def step():
        seq, starts, slots, left, status = paged_plan(cached, new, table, free, count, block, 12)
        paged_append(k, v, slots, kc, vc, ks, vs)
        out, lse = paged_attention(q, kc, vc, ks, vs, table, seq, starts, 12)
        cached.copy_(seq)
        count.copy_(left)
        return out, lse, starts, slots

    step()  # warm-up with no new tokens
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, starts, slots = step()
    lens = [0, 0, 0]
    for turn, n in enumerate([[5, 0, 7], [1, 1, 1], [0, 11, 1], [4, 4, 4], [1, 1, 1]]):
        new.copy_(i32(n))
        for i, t in enumerate((k, v, q)):
            t.copy_(values(tuple(t.shape), BF16, 100 * turn + i))
        before = [t.cpu() for t in (kc, vc, ks, vs)]
        graph.replay()
        lens = [a + b for a, b in zip(lens, n)]
        s = slots.tolist()
        after = [t.cpu() for t in (kc, vc, ks, vs)]
        for x, c0, s0, c1, s1 in ((k, before[0], before[2], after[0], after[2]), (v, before[1], before[3], after[1], after[3])):
            want, scale = ref.append(x.cpu(), s, c0, s0)
            assert torch.equal(c1.double(), want) and torch.equal(s1.double(), scale)
        want, wlse, weight = ref.attention(q.cpu(), *after, table.tolist(), lens, starts.tolist())
        assert ((out.cpu().double() - want).abs() <= ref.out_bound(want, weight, wlse, BF16, max(lens))).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,D,block", [(16, 2, 128, 16), (4, 1, 64, 32)])
def test_attention_chunks(kernel, dtype, H, Hkv, D, block):
    """Chunks of many rows a K/V head, whole prompts among them."""
    check(problem([300, 131, 517], [97, 131, 1], H, Hkv, D, block, dtype, seed=11), kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_nan_in_later_tokens(kernel, dtype, D):
    """A key that only later tokens of the step see holds NaN: they get NaN where it stands, the earlier ones nothing of it."""
    needs(kernel, dtype)
    q, kc, vc, ks, vs, table, lens, starts = problem([150, 40], [6, 5], 6, 2, D, 16, dtype, seed=12)
    args = lambda k, v: [q.cuda(), k.cuda(), v.cuda(), ks.cuda(), vs.cuda(), i32(table), i32(lens), i32(starts), 6, True, 0.0, kernel]  # noqa: E731
    clean, _ = pmkl_pytorch_ext.paged_attention_fw(*args(kc, vc))
    # request 0: row 148 (seen by its last two tokens); request 1: row 38, all of head 1
    bad = vc.clone()
    bad.view(torch.uint8)[table[0][148 // 16], 0, 148 % 16, 5] = 0x7F
    bad.view(torch.uint8)[table[0][148 // 16], 0, 148 % 16, D - 1] = 0xFF
    bad.view(torch.uint8)[table[1][38 // 16], 1, 38 % 16] = 0x7F
    out, lse = pmkl_pytorch_ext.paged_attention_fw(*args(kc, bad))
    want = torch.zeros(out.shape, dtype=torch.bool)
    want[4:6, 0:3, 5] = want[4:6, 0:3, D - 1] = True
    want[9:11, 3:6] = True
    assert torch.equal(out.isnan().cpu(), want)
    assert torch.equal(out[~want.cuda()], clean[~want.cuda()])
    # the same in the keys: whole rows
    bad = kc.clone()
    bad.view(torch.uint8)[table[0][148 // 16], 0, 148 % 16, 5] = 0x7F
    out, lse = pmkl_pytorch_ext.paged_attention_fw(*args(bad, vc))
    want = torch.zeros(out.shape, dtype=torch.bool)
    want[4:6, 0:3] = True
    assert torch.equal(out.isnan().cpu(), want) and torch.equal(lse.isnan().cpu(), want[:, :, 0])


@pytest.mark.parametrize("kernel", KERNELS)
def test_attention_keys_and_values_in_different_layouts(kernel):
    prob = list(problem([70, 200], [2, 1], 4, 2, 64, 16, F16, seed=13))
    prob[1] = prob[1].transpose(1, 2).contiguous().transpose(1, 2)  # keys: rows outside the heads
    big = torch.zeros(prob[2].shape[0], 2, 16, 2 * 64, dtype=torch.uint8)  # values: every other 64 bytes of a row
    big[..., 64:] = prob[2].view(torch.uint8)
    prob[2] = big.view(torch.float8_e4m3fn)[..., 64:]
    check(tuple(prob), kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("D,rows_first", [(128, False), (64, True)])
def test_cache_past_32_bit_offsets(kernel, D, rows_first):
    """Pages whose bytes lie past 2^32: written by paged_append and read back by the attention, against a small cache."""
    Hkv, block = 4, 64
    pages = (9 << 29) // (Hkv * block * D)  # 4.5 GiB
    shape = (pages, block, Hkv, D) if rows_first else (pages, Hkv, block, D)
    cache = torch.empty(shape, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    cache = cache.transpose(1, 2) if rows_first else cache
    scale = torch.ones(pages, Hkv, device="cuda")
    x = values((150, Hkv, D), BF16, 14)
    far = [pages - 1, 3, pages - 2]
    slots = torch.tensor([p * block + i for p in far for i in range(block)][:150], device="cuda")
    paged_append(x, x, slots, cache, cache, scale, scale)  # keys and values share one cache here
    near, near_scale = torch.zeros(3, Hkv, block, D, device="cuda").to(torch.float8_e4m3fn), torch.ones(3, Hkv, device="cuda")
    paged_append(x, x, torch.arange(150, device="cuda"), near, near, near_scale, near_scale)
    q = values((2, 8, D), BF16, 15)
    a = pmkl_pytorch_ext.paged_attention_fw(q, cache, cache, scale, scale, i32([far]), i32([150]), i32([0, 2]), 2, True, 0.0, kernel)
    b = pmkl_pytorch_ext.paged_attention_fw(q, near, near, near_scale, near_scale, i32([[0, 1, 2]]), i32([150]), i32([0, 2]), 2,
                                            True, 0.0, kernel)
    for got, want in zip(a, b):
        assert torch.equal(got, want) and got.isfinite().all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_many_requests(kernel, dtype):
    """More requests than a CTA has threads, most of them short, some empty."""
    r = random.Random(16)
    lens = [r.choice([0, 1, 5, 16, 40]) for _ in range(600)] + [700]
    news = [r.choice([0, 1, 1, 2]) for _ in lens]
    check(problem(lens, news, 2, 1, 64, 16, dtype, seed=17), kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("H,Hkv,D", [(4, 2, 64), (4, 1, 128)])
def test_attention_zero_queries_over_zero_keys(kernel, dtype, H, Hkv, D):
    """Zero keys, appended (their pages get the smallest scale), under zero and other queries: the mean of the values."""
    block, lens, news = 16, [1, 17, 129, 160, 40], [1, 1, 1, 5, 40]
    width = max(-(-n // block) for n in lens)
    table, slots, pages = [], [], 0
    for n in lens:
        k = -(-n // block)
        table.append([pages + j for j in range(k)] + [-1] * (width - k))
        slots += [pages * block + i for i in range(n)]
        pages += k
    kc, vc = (torch.zeros(pages, Hkv, block, D, device="cuda").to(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = torch.ones(pages, Hkv, device="cuda"), torch.ones(pages, Hkv, device="cuda")
    paged_append(torch.zeros(len(slots), Hkv, D, device="cuda", dtype=dtype), values((len(slots), Hkv, D), dtype, 20),
                 torch.tensor(slots, device="cuda"), kc, vc, ks, vs)
    assert (ks == 2.0 ** -64).all()
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    q = torch.zeros(starts[-1], H, D, dtype=dtype)
    q[:, 1] = values((starts[-1], D), dtype, 21).cpu()
    check((q, kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table, lens, starts), kernel=kernel)
    check((q, kc.cpu(), vc.cpu(), ks.cpu(), vs.cpu(), table, lens, starts), kernel=kernel, scale=1e-30)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_small_queries_over_large_keys(kernel, dtype):
    """Queries near 2^-66 over keys near 2^66, near 2^50 over 2^-50: ordinary scores; keys of scale 0 are keys of 0."""
    q, kc, vc, ks, vs, table, lens, starts = problem([700, 90], [1, 5], 4, 2, 128, 16, dtype, seed=26)
    check((q * 2.0 ** -66, kc, vc, ks * 2.0 ** 66, vs, table, lens, starts), kernel=kernel)
    check((q * 2.0 ** 50, kc, vc, ks * 2.0 ** -50, vs, table, lens, starts), kernel=kernel)
    check((q, kc, vc, torch.where(ks.isnan(), ks, 0.0), vs, table, lens, starts), kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_one_strong_key_over_many_weak(kernel, dtype, D):
    """One key of value zero, 19 nats above 64 Ki others: what is left of the output is theirs.

    A weight is rounded against the largest one at 2^7 (16-bit queries; 2^13 with
    fp32 queries, in two parts): 2^-25 at the lower end of fp16, so 2^-32 (2^-38)
    of the largest value a key, beside the relative errors that out_bound has."""
    needs(kernel, dtype, D)
    block, n, batch = 128, 1 << 16, 300  # (as many requests as CTAs: a CTA sees a request whole)
    g = torch.Generator().manual_seed(22)
    pages = n // block
    k = torch.zeros(pages, 1, block, D)
    k[:, 0, :, 1] = torch.randn(pages, block, generator=g)
    v = 1 + 0.25 * torch.randn(pages, 1, block, D, generator=g)
    k[6, 0, 9, 0], k[6, 0, 9, 1], v[6, 0, 9] = 8.0, 0.0, 0.0
    kc, vc = k.to(torch.float8_e4m3fn), v.to(torch.float8_e4m3fn)
    ones = torch.ones(pages, 1)
    q = torch.zeros(1, 1, D)
    q[0, 0, 0], q[0, 0, 1] = 19.0, 4.0
    q = q.to(dtype)
    order = list(range(pages))
    want, lse, weight = ref.attention(q, kc, vc, ones, ones, [order], [n], [0, 1], scale=0.125)
    table = i32([order, order[::-1]]).repeat(batch // 2, 1)  # the strong key early and late
    out, got_lse = pmkl_pytorch_ext.paged_attention_fw(
        q.cuda().repeat(batch, 1, 1), kc.cuda(), vc.cuda(), ones.cuda(), ones.cuda(), table, i32([n] * batch), None, 1, True,
        0.125, kernel)
    rel, floor = (2.0 ** -20, 2.0 ** -38) if dtype == F32 else (2.0 ** -11, 2.0 ** -32)
    bound = (rel + 2.0 ** -15) * weight + n * floor * float(vc.float().abs().max()) + 0.5 * ref.ulp(want, dtype)
    err = (out.cpu().double() - want).abs()
    assert (err <= bound).all(), f"err {err.max():.3e} of {float(want.abs().max()):.3e}, worst err / bound {(err / bound).max():.3f}"
    assert ((got_lse.cpu().double() - lse).abs() <= ref.lse_bound(lse)).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype,exponent,key_exponent", [(F32, 103, 0), (F32, 122, 0), (F32, 23, 6), (F16, 14, 30), (BF16, 103, 0),
                                                         (BF16, 27, 4)])
def test_attention_scores_far_from_zero(kernel, dtype, exponent, key_exponent):
    """Scores of both signs between 1e9 and 1e38, where one key (or three equal ones of a page) leads by an eighth.

    fp32 scores of this size differ by more than their rounding or not at all, so
    the output is the leaders' mean; lse is off by their relative rounding, 2^-15
    at most."""
    needs(kernel, dtype)
    q, kc, vc, ks, vs, table, lens, starts = problem([1, 3, 200], [1, 1, 20], 2, 1, 64, 16, dtype, seed=23)
    kc = torch.where(kc.view(torch.uint8) == 0x7F, kc.view(torch.uint8), 0x38)  # ones where written
    kc[table[2][77 // 16], 0, 77 % 16] = 0x39  # 1.125
    kc[table[2][101 // 16], 0, 101 % 16] = 0x36  # 0.875
    kc, ks = kc.view(torch.float8_e4m3fn), torch.where(ks.isnan(), ks, 2.0 ** key_exponent)
    for sign in (1, -1):
        q = torch.full_like(q, sign * 2.0 ** exponent)
        want, lse, weight = ref.attention(q, kc, vc, ks, vs, table, lens, starts)
        out, got = pmkl_pytorch_ext.paged_attention_fw(q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), i32(table), i32(lens),
                                                       i32(starts), 20, True, 0.0, kernel)
        assert ((out.cpu().double() - want).abs() <= ref.out_bound(want, weight, lse, dtype, 200)).all()
        assert ((got.cpu().double() - lse).abs() <= 2.0 ** -15 * lse.abs()).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("low,high", [(-64, 64), (-64, 20), (-20, 64)])
def test_attention_value_scales_at_the_ends_of_their_range(kernel, dtype, low, high):
    """Pages of values at both ends of 2^-64 .. 2^64: each key counts in the sum, whatever its page's scale."""
    for seed in range(3):
        prob = problem([700, 33, 1500, 257], [1, 1, 2, 40], 4, 2, 128, 16, dtype, seed=30 + seed)
        vs = prob[4]
        g = torch.Generator().manual_seed(seed)
        vs.copy_(torch.where(vs.isnan(), vs, torch.exp2(torch.where(torch.rand(vs.shape, generator=g) < 0.5, low, high).float())))
        check(prob, kernel=kernel)


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hint", [0, 1, 3, 70, 1 << 20])
def test_attention_writes_every_row(kernel, dtype, hint):
    """Whatever max_query_len says: rows past it, before the first request and behind the last one."""
    needs(kernel, dtype)
    for H, Hkv, D in ((4, 4, 64), (8, 1, 128)):
        q, kc, vc, ks, vs, table, lens, starts = problem([64, 1, 200, 90], [3, 1, 33, 70], H, Hkv, D, 16, dtype, seed=24, tail=9)
        starts = [s + 4 for s in starts]
        want, lse, weight = ref.attention(q, kc, vc, ks, vs, table, lens, starts)
        dev = [t.cuda() for t in (q, kc, vc, ks, vs)] + [i32(table), i32(lens), i32(starts)]
        stale = [torch.full((n,), math.nan, device="cuda") for n in (q.numel(), q.numel() // 2, q.numel() // D)]
        del stale  # (memory that the outputs are likely to get)
        out, got_lse = pmkl_pytorch_ext.paged_attention_fw(*dev, hint, True, 0.0, kernel)
        assert ((out.cpu().double() - want).abs() <= ref.out_bound(want, weight, lse, dtype, max(lens))).all()
        empty, l = lse.isinf(), got_lse.cpu().double()
        assert torch.equal(l.isinf(), empty) and (l[empty] < 0).all()
        assert ((l - lse).abs()[~empty] <= ref.lse_bound(lse)[~empty]).all()


def test_attention_without_max_query_len():
    """The function's default covers a prompt."""
    q, kc, vc, ks, vs, table, lens, starts = problem([64, 90], [33, 70], 4, 2, 64, 16, BF16, seed=25)
    dev = [t.cuda() for t in (q, kc, vc, ks, vs)] + [i32(table), i32(lens)]
    out, lse = paged_attention(*dev, i32(starts))
    named, named_lse = paged_attention(*dev, query_starts=i32(starts), max_query_len=70)
    want, want_lse, weight = ref.attention(q, kc, vc, ks, vs, table, lens, starts)
    for o, l in ((out, lse), (named, named_lse)):
        assert ((o.cpu().double() - want).abs() <= ref.out_bound(want, weight, want_lse, BF16, 90)).all()
        assert ((l.cpu().double() - want_lse).abs() <= ref.lse_bound(want_lse)).all()


# ---------------------------------------------------------------- refusals
def test_refusals():
    q, kc, vc, ks, vs, table, lens, starts = problem([20], [1], 4, 2, 64, 16, F16, seed=8)
    q, kc, vc, ks, vs, t, n = q.cuda(), kc.cuda(), vc.cuda(), ks.cuda(), vs.cuda(), i32(table), i32(lens)
    ok = (q, kc, vc, ks, vs, t, n)
    paged_attention(*ok)

    def refused(match, *args, **kw):
        with pytest.raises(RuntimeError, match=match):
            paged_attention(*args, **kw)

    refused("dtype|tensor", q.double(), *ok[1:])
    refused("hidden size", q[..., :32], *ok[1:])
    refused("hidden size", q[:, :3], *ok[1:])
    refused("same shape", q, kc, vc[:, :1], ks, vs[:, :1].contiguous(), t, n)
    refused("float8", q, kc.float(), *ok[2:])
    refused("k_scale", q, kc, vc, ks.half(), vs, t, n)
    refused("k_scale", q, kc, vc, ks[:1], vs, t, n)
    refused("block_table", q, kc, vc, ks, vs, t.long(), n)
    refused("block_table", q, kc, vc, ks, vs, t.repeat(2, 1), n)
    refused("seq_lens", q, kc, vc, ks, vs, t, n.long())
    refused("query_starts", *ok, query_starts=i32([0]))
    refused("one token", q.repeat(2, 1, 1), *ok[1:])
    refused("max_query_len", *ok, max_query_len=-1)
    refused("on cuda", q, kc, vc, ks, vs, t, n.cpu())
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        pmkl_pytorch_ext.paged_attention_fw(*ok, None, 1, True, 0.0, 99)
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        wide = torch.zeros(1, 1, 16, 300, device="cuda").to(torch.float8_e4m3fn)
        one = torch.ones(1, 1, device="cuda")
        paged_attention(torch.zeros(1, 1, 300, device="cuda"), wide, wide, one, one, t, n)
    k = torch.zeros(3, 2, 64, device="cuda", dtype=F16)
    slots = torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in ((k[:, :1], k, slots), (k, k.float(), slots), (k, k, slots[:2]), (k, k, slots.int()), (k[..., :32], k[..., :32], slots)):
        with pytest.raises(RuntimeError):
            paged_append(*bad, kc, vc, ks, vs)
    for bad in ((i32([1]), i32([1, 2]), 16, 8), (i32([1]), i32([1]), 0, 8), (i32([1]), i32([1]), 16, -1), (n.long(), n, 16, 8)):
        with pytest.raises(RuntimeError):
            paged_plan(bad[0], bad[1], t, i32([1]), i32([1]), bad[2], bad[3])


def test_example_runs():
    import subprocess
    import sys
    from pathlib import Path

    example = Path(__file__).resolve().parent.parent / "examples" / "paged_decode.py"
    out = subprocess.run([sys.executable, str(example), "--steps", "12", "--check"], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert "12 steps" in out.stdout
