"""The token-step operators (include/hipvoc_ops.h) on an MI355X against plain 64-bit implementations.

Tolerances count roundings: a value rounded to a type is off by at most finfo.eps / 2 of itself (u(t) below), an operation in 32 bits by
2^-24 of its result, so a sum of n terms in any order by n * 2^-24 of the sum of their magnitudes."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

ACT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STORE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}
U32 = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.fixture(scope="module")
def ops(pkg):
    torch.cuda.init()
    o = pkg.HipOps.open(0)
    yield o
    o.sync()
    o.close()


def rnd(shape, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * spread).to(dtype)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def encode(x, store):
    """Codes and scales of [..., n] as the header defines them, in numpy's 32-bit arithmetic (CPU)."""
    x = x.float().numpy()
    scale = np.abs(x).max(-1) * (np.float32(1) / np.float32(TOP[store]))
    assert scale.dtype == np.float32
    with np.errstate(divide="ignore", invalid="ignore"):
        q = np.where(scale[..., None] > 0, x / scale[..., None], np.float32(0)).astype(np.float32)
    codes = torch.from_numpy(np.rint(q)).to(torch.int8) if store == "int8" else torch.from_numpy(q).to(torch.float8_e4m3fn)
    return codes, torch.from_numpy(scale)


class Paged:
    """A cache on the GPU whose unused places hold NaN (codes: the largest), and the plain values of its sequences on the CPU."""

    def __init__(self, ops, lens, kv, hd, page, act, store="same", seed=0, extra_pages=3, width=None, together=False, spread=1.0):
        self.lens, self.act, self.store, self.kv, self.hd, self.page = list(lens), ACT[act], store, kv, hd, page
        need = [-(-n // page) for n in lens]
        self.width = max(need + [1]) if width is None else width
        n_pages = sum(need) + extra_pages
        order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed + 9)).tolist()
        table = torch.full((len(lens), self.width), -7, dtype=torch.int32)             # entries that no token needs are garbage
        st = self.act if store == "same" else STORE[store]
        shape = (n_pages, kv, page, hd)
        if store == "same":
            pool = [torch.full(shape, float("nan"), dtype=st) for _ in range(2)]
            scales = [None, None]
        else:
            pool = [torch.full(shape, 127, dtype=torch.uint8).view(st) for _ in range(2)]     # e4m3: NaN
            scales = [torch.full(shape[:3], float("nan")) for _ in range(2)]
        self.k, self.v = [], []
        at = 0
        for b, n in enumerate(lens):
            pages = order[at:at + need[b]]
            at += need[b]
            table[b, :need[b]] = torch.tensor(pages, dtype=torch.int32)
            for i, mine in enumerate((self.k, self.v)):
                x = rnd((n, kv, hd), self.act, seed * 1000 + 10 * b + i, spread if i == 0 else 1.0)
                if store == "same":
                    codes, value = x, x.double()
                else:
                    codes, sc = encode(x, store) if n else (torch.zeros((0, kv, hd), dtype=st), torch.zeros((0, kv)))
                    value = codes.double() * sc.double()[..., None]
                mine.append(value)
                for j, p in enumerate(pages):
                    m = min(page, n - j * page)
                    dst = pool[i].view(torch.uint8) if store == "e4m3" else pool[i]
                    src = codes[j * page:j * page + m].transpose(0, 1)
                    dst[p, :, :m] = src.contiguous().view(torch.uint8) if store == "e4m3" else src
                    if store != "same":
                        scales[i][p, :, :m] = sc[j * page:j * page + m].t()
        if together:                                                              # K and V as halves of one allocation
            both = torch.stack(pool, 1).cuda() if store != "e4m3" else torch.stack([p.view(torch.uint8) for p in pool], 1).cuda().view(st)
            gk, gv = both[:, 0], both[:, 1]
        else:
            gk, gv = [p.cuda() for p in pool]
        self.cache = ops.kv_cache(gk, gv, *[s.cuda() if s is not None else None for s in scales])
        self.table = table.cuda()
        self.lens_dev = ints(self.lens)


def attention_ref(P, q, scale, window):
    """(out, lse, bound of out's error, bound of lse's error) in 64 bits."""
    b, heads, hd = q.shape
    outs, lses, bo, bl = [], [], [], []
    rep = heads // P.kv
    # the weights' rounding for the product with V: two f16 or two bf16, the second holding what the first leaves over
    p16 = 0.0 if P.act == torch.float32 else u(torch.float16 if P.act == torch.float16 and P.store == "same" else torch.bfloat16) ** 2
    for s in range(b):
        n = P.lens[s]
        lo = max(0, n - window) if window else 0
        if n == 0:
            outs.append(torch.zeros(heads, hd, dtype=torch.float64)); lses.append(torch.full((heads,), -math.inf, dtype=torch.float64))
            bo.append(torch.zeros(heads, hd, dtype=torch.float64)); bl.append(torch.zeros(heads, dtype=torch.float64))
            continue
        k = P.k[s][lo:n].repeat_interleave(rep, 1).permute(1, 0, 2)            # [heads, n, hd]
        v = P.v[s][lo:n].repeat_interleave(rep, 1).permute(1, 0, 2)
        qq = q[s].double()[:, None]
        score = (k * qq).sum(-1) * scale
        mag = (k.abs() * qq.abs()).sum(-1) * abs(scale)
        # a score: hd products and sums, two multiplications (scale, code's scale), one conversion to powers of two; then 2^x and its argument
        delta = ((hd + 8) * U32 * mag + 8 * U32 * (1 + score.abs())).amax(-1) + 2.0 ** -21
        w = torch.softmax(score, -1)
        out = (w[..., None] * v).sum(1)
        wv = (w[..., None] * v.abs()).sum(1)
        m = n - lo
        err = wv * (2 * delta[:, None] + p16 + (2 * m + 16) * U32)
        if P.act == torch.float16 and P.store == "same":
            # weights below the type's normal range (the largest weight being 2^15 there) are off by half its smallest step
            err = err + w.amax(-1)[:, None] * m * 2.0 ** -40 * v.abs().amax(1)
        outs.append(out)
        bo.append(err + u(P.act) * (out.abs() + err) + 2.0 ** -24 * (P.act == torch.float16))
        lse = torch.logsumexp(score, -1)
        lses.append(lse)
        bl.append(delta + m * U32 + 8 * U32 * (1 + lse.abs()))
    return torch.stack(outs), torch.stack(lses), torch.stack(bo), torch.stack(bl)


def check_attention(ops, P, q, scale=None, window=0, max_len=None, **kw):
    hd = q.shape[-1]
    out, lse = ops.attention(q.cuda() if not q.is_cuda else q, P.cache, P.table, P.lens_dev, scale=scale, window=window, max_len=max_len, lse=True, **kw)
    ops.sync()
    ro, rl, bo, bl = attention_ref(P, q.cpu(), 1 / math.sqrt(hd) if scale is None else scale, window)
    d = (out.cpu().double() - ro).abs()
    assert bool((d <= bo).all()), f"out off by up to {float((d / bo.clamp_min(1e-300)).max()):.3g} of its bound, at {np.unravel_index(int((d - bo).argmax()), d.shape)}"
    empty = torch.tensor([n == 0 for n in P.lens])
    got = lse.cpu().double()
    assert bool((got[empty] == -math.inf).all())
    d = (got[~empty] - rl[~empty]).abs()
    assert bool((d <= bl[~empty]).all()), float((d / bl[~empty]).max())
    return out, lse


# ---------------------------------------------------------------------------------------------------------------------
# the cache
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("kv,hd,page", [(1, 64, 8), (3, 128, 16), (8, 64, 256), (20, 128, 8), (33, 64, 8)])
def test_kv_write_and_read(ops, act, store, kv, hd, page):
    """Codes and scales bit for bit, the values read back bit for bit, unwritten places and padding rows untouched."""
    P = Paged(ops, [0, 5, page + 3, 1], kv, hd, page, act, store, seed=3, width=4)
    past, new = [0, 5, page + 3, 1], [1, page, 0, 2 * page + 1]
    table = torch.randperm(16, generator=torch.Generator().manual_seed(1)).to(torch.int32).reshape(4, 4)
    shape = (17, kv, page, hd)
    st = ACT[act] if store == "same" else STORE[store]
    raw = torch.full((17 * kv * page * hd * torch.tensor([], dtype=st).element_size(),), 0x55, dtype=torch.uint8)
    k, v = raw.clone().cuda().view(st).reshape(shape), raw.clone().cuda().view(st).reshape(shape)
    ks = vs = None
    if store != "same":
        ks, vs = torch.full(shape[:3], 9.0, device="cuda"), torch.full(shape[:3], 9.0, device="cuda")
    cache = ops.kv_cache(k, v, ks, vs)
    rows = sum(new)
    x = [rnd((rows + 5, kv, hd), ACT[act], 20 + i, 3.0) for i in range(2)]
    x[0][1, 0] = 0                                             # a row of zeros
    x[1][2, kv - 1] *= 1e-3
    cu = [sum(new[:i]) for i in range(5)]
    ops.kv_write(cache, x[0].cuda(), x[1].cuda(), table.cuda(), ints(cu), ints(past))
    ops.sync()
    want = [raw.clone().view(st).reshape(shape), raw.clone().view(st).reshape(shape)]
    wsc = [torch.full(shape[:3], 9.0), torch.full(shape[:3], 9.0)]
    as8 = lambda t: t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t  # noqa: E731
    for i in range(2):
        codes, sc = (x[i], None) if store == "same" else encode(x[i], store)
        for b in range(4):
            for j in range(new[b]):
                p = past[b] + j
                pg, at = int(table[b, p // page]), p % page
                as8(want[i])[pg, :, at] = as8(codes[cu[b] + j])
                if sc is not None:
                    wsc[i][pg, :, at] = sc[cu[b] + j]
    for i, got in enumerate((k, v)):
        assert torch.equal(got.cpu().view(torch.uint8), want[i].view(torch.uint8))
        if store != "same":
            assert torch.equal((ks, vs)[i].cpu(), wsc[i])
    # read the new rows back, into strided tensors with padding behind them
    big = [torch.full((rows + 3, 2 * kv, hd), 7.0, dtype=ACT[act], device="cuda") for _ in range(2)]
    ops.kv_read(cache, table.cuda(), ints(cu), ints(past), rows + 3, out=(big[0][:, :kv], big[1][:, kv:]))
    ops.sync()
    for i in range(2):
        got = (big[0][:, :kv], big[1][:, kv:])[i].cpu()
        codes, sc = (x[i], None) if store == "same" else encode(x[i], store)
        value = codes[:rows] if sc is None else (codes[:rows].float() * sc[:rows, :, None]).to(ACT[act])
        assert torch.equal(got[:rows], value)
        assert bool((got[rows:] == 7).all())
        other = (big[0][:, kv:], big[1][:, :kv])[i].cpu()
        assert bool((other == 7).all())


def test_kv_many_sequences_and_empty_calls(ops):
    """More sequences than a wave has lanes, most of them empty; calls with no rows or no sequences."""
    n, kv, hd, page = 200, 2, 64, 8
    new = [(i * 7) % 4 if i % 3 else 0 for i in range(n)]
    cu = np.concatenate([[0], np.cumsum(new)]).tolist()
    k = torch.zeros((n, kv, page, hd), dtype=torch.float32, device="cuda")
    v = torch.zeros_like(k)
    cache = ops.kv_cache(k, v)
    table = torch.arange(n, dtype=torch.int32).flip(0).reshape(n, 1).cuda()
    x, y = rnd((cu[-1], kv, hd), torch.float32, 1), rnd((cu[-1], kv, hd), torch.float32, 2)
    ops.kv_write(cache, x.cuda(), y.cuda(), table, ints(cu), ints([i % 5 for i in range(n)]))
    gx, gy = ops.kv_read(cache, table, ints(cu), ints([i % 5 for i in range(n)]), cu[-1])
    ops.sync()
    assert torch.equal(gx.cpu(), x) and torch.equal(gy.cpu(), y)
    assert int((k.cpu() != 0).any(-1).sum()) == cu[-1] * kv
    empty = x[:0].cuda()
    ops.kv_write(cache, empty, empty, table, ints(cu), ints([0] * n))
    a, b = ops.kv_read(cache, table[:0], ints([0]), ints([]), 3)
    assert a.shape == (3, kv, hd)
    ops.sync()


def test_kv_special_values(ops):
    """Rows with an infinity or NaN read back as NaN, their neighbours are untouched; subnormal and largest rows keep their scale's accuracy."""
    kv, hd = 1, 64
    x = rnd((6, kv, hd), torch.float32, 4)
    x[1, 0, 3] = math.inf
    x[2, 0, 7] = math.nan
    x[3] *= 1e-42
    x[4] = 3e38 * torch.sign(x[4])
    x[5] *= 1e-37
    for store in ("int8", "e4m3"):
        k = torch.zeros((1, kv, 8, hd), dtype=torch.uint8, device="cuda").view(STORE[store])
        s = torch.zeros((1, kv, 8), device="cuda")
        cache = ops.kv_cache(k, k.clone(), s, s.clone())
        ops.kv_write(cache, x.cuda(), x.cuda(), ints([[0]]), ints([0, 6]), ints([0]))
        got, _ = ops.kv_read(cache, ints([[0]]), ints([0, 6]), ints([0]), 6, dtype=torch.float32)
        ops.sync()
        got = got.cpu()
        assert bool(got[1].isnan().all()) and bool(got[2].isnan().all())
        step = 0.5 if store == "int8" else 16.0                  # half a step of the largest codes
        for r in (0, 4, 5):
            top = float(x[r].abs().max())
            assert float((got[r] - x[r]).abs().max()) <= top / TOP[store] * step * (1 + 2.0 ** -20)
        # the scale of a subnormal row is itself a subnormal of few bits: off by half of 2^-149, times a code of up to TOP
        top = float(x[3].abs().max())
        assert float((got[3] - x[3]).abs().max()) <= top / TOP[store] * step + (TOP[store] + step) * 2.0 ** -150 + 2.0 ** -149


def test_kv_deferred_errors(pkg, ops):
    """Pages and positions out of range are not followed: nothing else is written, such rows read as NaN, sync() says so once."""
    kv, hd, page = 2, 64, 8
    k = torch.zeros((2, kv, page, hd), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    cache = ops.kv_cache(k, v)
    x = rnd((4, kv, hd), torch.bfloat16, 1).cuda()
    for table, first in [([[2]], [0]), ([[-1]], [0]), ([[2 ** 31 - 1]], [3]), ([[0]], [-1 - 2 ** 20]), ([[0]], [8]), ([[0]], [2 ** 31 - 2])]:
        ops.kv_write(cache, x, x, ints(table), ints([0, 4]), ints(first))
        with pytest.raises(pkg.HipVocError) as e:
            ops.sync()
        assert e.value.code == -2
        ops.sync()
        assert not bool(k.any()) and not bool(v.any())
        a, b = ops.kv_read(cache, ints(table), ints([0, 4]), ints(first), 4)
        with pytest.raises(pkg.HipVocError):
            ops.sync()
        assert bool(a.isnan().all()) and bool(b.isnan().all())
    # half of the rows are sound: they are written, the rest is not
    ops.kv_write(cache, x, x, ints([[1]]), ints([0, 4]), ints([6]))
    with pytest.raises(pkg.HipVocError):
        ops.sync()
    assert torch.equal(k[1, :, 6:].transpose(0, 1), x[:2]) and not bool(k[0].any()) and not bool(k[1, :, :6].any())


# ---------------------------------------------------------------------------------------------------------------------
# attention
LENS = [0, 1, 7, 8, 31, 32, 33, 64, 100, 127, 128, 129, 255, 256, 257, 300]


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,rep,page", [(1, 1, 8), (2, 2, 16), (3, 4, 32), (1, 7, 256), (2, 17, 64)])
def test_attention_lengths(ops, act, store, hd, kv, rep, page):
    P = Paged(ops, LENS, kv, hd, page, act, store, seed=kv * 10 + rep)
    q = rnd((len(LENS), kv * rep, hd), ACT[act], 5)
    check_attention(ops, P, q)
    check_attention(ops, P, q, max_len=300)


@pytest.mark.parametrize("act,store", [("f32", "same"), ("f16", "same"), ("bf16", "int8"), ("f16", "e4m3"), ("f32", "int8")])
@pytest.mark.parametrize("window", [1, 5, 31, 32, 33, 72, 256, 5000])
def test_attention_window(ops, act, store, window):
    """A window hides all but the last tokens: 72 is the decoder transformer's."""
    P = Paged(ops, [0, 1, 40, 72, 73, 300, 1031], 2, 64, 16, act, store, seed=window)
    check_attention(ops, P, rnd((7, 6, 64), ACT[act], 6), window=window)


@pytest.mark.parametrize("act,store,hd,rep", [("bf16", "same", 128, 4), ("f16", "int8", 64, 3), ("f32", "same", 64, 2), ("bf16", "e4m3", 128, 8), ("f32", "e4m3", 128, 1)])
def test_attention_split_and_joined(ops, act, store, hd, rep):
    """Long sequences in many chunks beside short ones in few, and a bound far above the lengths."""
    P = Paged(ops, [5003, 1, 0, 2048, 777], 1, hd, 64, act, store, seed=2, width=160)
    q = rnd((5, rep, hd), ACT[act], 7, 2.0)
    a = check_attention(ops, P, q, max_len=5003)
    b = check_attention(ops, P, q)                              # 160 pages: 10240 positions
    again = check_attention(ops, P, q, max_len=5003)
    assert torch.equal(a[0], again[0]) and torch.equal(a[1], again[1])         # the order of every sum is fixed
    assert b[0].shape == a[0].shape
    check_attention(ops, P, q, max_len=5003, window=3000)


# bounds over 768 keys (1024 with 256 key heads or more in the call): the tiles of all sequences are shared out over the card
@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kv,rep,page", [(1, 1, 8), (2, 2, 16), (3, 4, 256), (1, 17, 64), (2, 8, 32)])
def test_attention_shared_out(ops, act, store, hd, kv, rep, page):
    """Empty and short sequences among long ones, so that a wave's share has many pieces; windows that are short, long and over the bound."""
    P = Paged(ops, [0, 1, 33, 800, 0, 0, 5, 64, 1500, 31, 300, 0], kv, hd, page, act, store, seed=kv * 10 + rep, together=page == 16)
    q = rnd((12, kv * rep, hd), ACT[act], 5)
    check_attention(ops, P, q)
    check_attention(ops, P, q, window=781)
    check_attention(ops, P, q, window=4000)


@pytest.mark.parametrize("act,store", [("f32", "same"), ("bf16", "int8"), ("f16", "same")])
@pytest.mark.parametrize("n", [1023, 1024, 1025])
def test_attention_many_sequences(ops, act, store, n):
    """As many sequences as a workgroup adds up, and one more: those are not cut."""
    lens = [(i * 37) % 90 for i in range(n)]
    lens[n // 2], lens[-1] = 1100, 77
    P = Paged(ops, lens, 1, 64, 16, act, store, seed=n)
    check_attention(ops, P, rnd((n, 2, 64), ACT[act], 3))


def test_attention_all_empty(ops):
    for lens, bound in (([0, 0, 0], None), ([0], 0), ([0, 0], 5000)):
        P = Paged(ops, lens, 2, 64, 8, "bf16", seed=1, width=700)
        out, lse = ops.attention(torch.full((len(lens), 4, 64), 3.0, dtype=torch.bfloat16, device="cuda"), P.cache, P.table, P.lens_dev, max_len=bound, lse=True)
        ops.sync()
        assert not bool(out.any()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("act", ["f16", "bf16", "f32"])
def test_attention_many_small_weights(ops, act):
    """One key far above 40000 others, each of which has e^-16.25 of its weight, 1.47 * 2^-24: together they are the result."""
    n, page, less = 40001, 64, 16.25
    pages = -(-n // page)
    k = torch.zeros((pages, 1, page, 64), dtype=ACT[act], device="cuda")
    v = torch.ones_like(k)
    k[..., 0] = -less
    k[0, 0, 0], v[0, 0, 0] = 0, 0
    q = torch.zeros((1, 1, 64), dtype=ACT[act], device="cuda")
    q[..., 0] = 1
    table = torch.arange(pages, dtype=torch.int32, device="cuda")[None]
    out = ops.attention(q, ops.kv_cache(k, v), table, ints([n]), scale=1.0, max_len=n)
    ops.sync()
    p = (n - 1) * math.exp(-less)
    ref = p / (1 + p)
    delta = (64 + 8) * U32 * less + 8 * U32 * (1 + less) + 2.0 ** -21                  # as in attention_ref
    rel = 2 * delta + (2 * n + 16) * U32 + u(ACT[act]) + u(torch.bfloat16) ** 2
    assert float((out.cpu().double() - ref).abs().max()) <= rel * ref


def test_attention_lse_joins_two_caches(ops):
    """The log-sums put two halves of a context together: what lse is for."""
    P = Paged(ops, [90], 2, 64, 8, "f32", seed=4)
    A, B = Paged(ops, [40], 2, 64, 8, "f32", seed=5), Paged(ops, [50], 2, 64, 8, "f32", seed=6)
    P.k, P.v = [torch.cat([A.k[0], B.k[0]])], [torch.cat([A.v[0], B.v[0]])]
    q = rnd((1, 4, 64), torch.float32, 8)
    (oa, la), (ob, lb) = [ops.attention(q.cuda(), X.cache, X.table, X.lens_dev, lse=True) for X in (A, B)]
    lse = torch.logaddexp(la.double(), lb.double())
    out = oa.double() * (la.double() - lse).exp()[..., None] + ob.double() * (lb.double() - lse).exp()[..., None]
    ro, rl, bo, bl = attention_ref(P, q, 1 / 8, 0)
    assert bool(((out.cpu() - ro).abs() <= 4 * bo).all()) and bool(((lse.cpu() - rl).abs() <= 4 * bl).all())


@pytest.mark.parametrize("act", ["f32", "bf16", "f16"])
def test_attention_strided_and_scaled(ops, act):
    """q as a slice of a fused projection, out into a slice, K and V in one allocation, another scale, sharp and flat softmax."""
    P = Paged(ops, [50, 333], 2, 128, 16, act, seed=11, together=True, spread=4.0)
    fused = rnd((2, 12, 128), ACT[act], 9)
    fused = fused.cuda()
    q = fused[:, 3:11]
    into = torch.full((2, 10, 128), 5.0, dtype=ACT[act], device="cuda")
    for scale in (1.0, 0.001, -0.3, 0.0):
        out, _ = check_attention(ops, P, q, scale=scale, out=into[:, 1:9])
        assert out.data_ptr() == into[:, 1:9].data_ptr()
        assert bool((into[:, 0] == 5).all()) and bool((into[:, 9] == 5).all())


@pytest.mark.parametrize("act,store", [("f32", "same"), ("bf16", "same"), ("f16", "same"), ("bf16", "int8")])
def test_attention_masked_places_are_never_read(ops, act, store):
    """The cache's unused places hold NaN, unused scales NaN, unused table entries -7 (Paged): results are finite.  An infinity or NaN among
    the tokens that are seen reaches its own sequence and head only."""
    P = Paged(ops, [33, 40, 65], 2, 64, 8, act, store, seed=12)
    q = rnd((3, 4, 64), ACT[act], 10)
    out, _ = check_attention(ops, P, q)
    assert bool(out.isfinite().all())
    page = int(P.table[1, 2])
    (P.cache.v if store == "same" else P.cache.v_scale)[page, 1, 3] = math.nan          # sequence 1, position 19, key head 1
    bad = ops.attention(q.cuda(), P.cache, P.table, P.lens_dev)
    ops.sync()
    assert bool(bad[1, 2:].isnan().all())
    keep = torch.ones(3, 4, dtype=torch.bool)
    keep[1, 2:] = False
    assert torch.equal(bad[keep.cuda()], out[keep.cuda()])
    seen = ops.attention(q.cuda(), P.cache, P.table, P.lens_dev, window=20)             # positions 20 .. 39: the NaN is out of sight
    ops.sync()
    assert bool(seen.isfinite().all())


def test_attention_deferred_errors(pkg, ops):
    P = Paged(ops, [40, 20, 9], 2, 64, 8, "bf16", seed=13)
    q = rnd((3, 4, 64), torch.bfloat16, 10).cuda()
    good = ops.attention(q, P.cache, P.table, P.lens_dev)
    for page in (-1, P.cache.n_pages, 2 ** 31 - 1):
        table = P.table.clone()
        table[1, 1] = page
        for kw in ({}, {"max_len": 40}):
            out, lse = ops.attention(q, P.cache, table, P.lens_dev, lse=True, **kw)
            with pytest.raises(pkg.HipVocError) as e:
                ops.sync()
            assert e.value.code == -2 and "page" in str(e.value)
            assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all()) and torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    for n in (-1, 41, 2 ** 31 - 1):
        out, lse = ops.attention(q, P.cache, P.table, ints([40, n, 9]), lse=True, max_len=40)
        with pytest.raises(pkg.HipVocError) as e:
            ops.sync()
        assert "length" in str(e.value)
        assert bool(out[1].isnan().all()) and bool(lse[1].isnan().all()) and torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    # in chunks
    L = Paged(ops, [5000, 4000], 1, 64, 8, "bf16", seed=13)
    q = rnd((2, 2, 64), torch.bfloat16, 10).cuda()
    good = ops.attention(q, L.cache, L.table, L.lens_dev, max_len=5000)
    table = L.table.clone()
    table[0, 300] = L.cache.n_pages + 5
    out = ops.attention(q, L.cache, table, L.lens_dev, max_len=5000)
    with pytest.raises(pkg.HipVocError):
        ops.sync()
    assert bool(out[0].isnan().all()) and torch.equal(out[1], good[1])
    out, lse = ops.attention(q, L.cache, L.table, ints([5001, 4000]), max_len=5000, lse=True)
    with pytest.raises(pkg.HipVocError):
        ops.sync()
    assert bool(out[0].isnan().all()) and bool(lse[0].isnan().all())
    # the keys of a call are cut over all its sequences: without the first one's, the second's are added up in another order
    ro, _, bo, _ = attention_ref(L, q.cpu(), 1 / 8, 0)
    assert bool(((out[1].cpu().double() - ro[1]).abs() <= bo[1]).all())
    ops.sync()


def test_attention_past_32_bits(ops):
    """Pages that start past 2^31 elements (and past 2^32 bytes) of the cache."""
    kv, hd, page, n_pages = 8, 128, 256, 9000                   # 2.36e9 values
    k = torch.empty((n_pages, kv, page, hd), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    s = torch.ones((n_pages, kv, page), device="cuda")
    cache = ops.kv_cache(k, v, s, torch.ones_like(s))
    rows = rnd((300, kv, hd), torch.bfloat16, 3)
    table = ints([[n_pages - 1, n_pages - 2]])
    ops.kv_write(cache, rows.cuda(), rows.flip(0).cuda(), table, ints([0, 300]), ints([0]))
    gk, gv = ops.kv_read(cache, table, ints([0, 300]), ints([0]), 300, dtype=torch.bfloat16)
    P = Paged.__new__(Paged)
    P.lens, P.act, P.store, P.kv, P.hd, P.page = [300], torch.bfloat16, "int8", kv, hd, page
    P.cache, P.table, P.lens_dev = cache, table, ints([300])
    P.k, P.v = [], []
    for mine, x, got in ((P.k, rows, gk), (P.v, rows.flip(0), gv)):
        c, sc = encode(x, "int8")
        mine.append(c.double() * sc.double()[..., None])
        assert torch.equal(got.cpu(), (c.float() * sc[..., None]).to(torch.bfloat16))
    check_attention(ops, P, rnd((1, 16, hd), torch.bfloat16, 4))


# ---------------------------------------------------------------------------------------------------------------------
# norm
def check_norm(ops, x, w, r, eps, quant, group):
    rows, cols = x.shape
    act = x.dtype
    res = ops.add_rmsnorm(x.cuda(), w.cuda(), None if r is None else r.cuda(), eps=eps, quant=quant, group=group)
    ops.sync()
    s = x.double() if r is None else x.double() + r.double()
    if r is None:
        assert res[0] is None
    else:
        got = res[0].cpu().double()
        assert bool(((got - s).abs() <= (u(act) + 2 * U32) * s.abs() + 2.0 ** -25 * (act == torch.float16)).all())
    y = s / torch.sqrt((s * s).mean(-1, keepdim=True) + eps) * w.double()
    rel = (cols / 2 + 12) * U32                               # sum of cols squares under a root, two roundings of s and its square, root, quotient, two products
    if quant is None:
        d = (res[1].cpu().double() - y).abs()
        assert bool((d <= (u(act) + 2 * rel) * y.abs() + 2.0 ** -25 * (act == torch.float16) + 1e-45).all()), float((d / y.abs()).max())
        return res
    n = group or cols
    assert res[2].shape == (rows, cols // n)
    top = y.reshape(rows, -1, n).abs().amax(-1)
    sc = res[2].cpu().double()
    assert bool(((sc - top / TOP[quant]).abs() <= (rel + 4 * U32) * top / TOP[quant] + 2.0 ** -149).all())
    assert res[1].dtype == STORE[quant]
    back = (res[1].cpu().double().reshape(rows, -1, n) * sc[..., None])
    yy = y.reshape(rows, -1, n)
    err = rel * yy.abs() + (sc[..., None] * (0.5 + 127 * 4 * U32) if quant == "int8" else 2.0 ** -4 * yy.abs() * (1 + 2 * rel) + sc[..., None] * 2.0 ** -10)
    assert bool(((back - yy).abs() <= err * (1 + 1e-6) + 1e-44).all())
    return res


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("quant", [None, "int8", "e4m3"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (2, 72), (5, 64), (1, 512), (9, 1000), (4, 1024), (7, 1536), (2, 2056), (3, 4096), (2, 8192), (1, 32768), (2, 40000)])
def test_add_rmsnorm(ops, act, quant, rows, cols):
    x, r, w = rnd((rows, cols), ACT[act], 1), rnd((rows, cols), ACT[act], 2, 3.0), rnd((cols,), ACT[act], 3)
    check_norm(ops, x, w, r, 1e-5, quant, 0)
    check_norm(ops, x, w, None, 1e-6, quant, 0)
    for group in (32, 64, 128):
        if quant and cols % group == 0:
            check_norm(ops, x, w, r, 1e-5, quant, group)


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("quant", [None, "int8", "e4m3"])
@pytest.mark.parametrize("off,cols", [(1, 96), (3, 256), (0, 128)])
def test_add_rmsnorm_strides_and_alignment(ops, act, quant, off, cols):
    """Rows inside a wider tensor, from any element on: the odd ones take the kernel that has no wide accesses."""
    wide = rnd((6, cols + 40), ACT[act], 4).cuda()
    res = rnd((6, cols + 13), ACT[act], 5).cuda()
    x, r, w = wide[:, off:off + cols], res[:, off:off + cols], rnd((cols,), ACT[act], 6)
    a = ops.add_rmsnorm(x, w.cuda(), r, eps=1e-5, quant=quant, group=32 if quant else 0)
    b = check_norm(ops, x.cpu().contiguous(), w, r.cpu().contiguous(), 1e-5, quant, 32 if quant else 0)
    assert torch.equal(a[0], b[0])
    if quant is None:
        # the two kernels add up in different orders; each is within (u + 2 rel) |y| of the exact row (check_norm), so they are within twice that
        far = 2 * (u(ACT[act]) + 2 * (cols / 2 + 12) * U32) * b[1].double().abs() * 1.01 + 2.0 ** -24 * (act == "f16")
        assert bool(((a[1].double() - b[1].double()).abs() <= far).all())
    else:
        assert bool(((a[2] - b[2]).abs() <= 1e-4 * b[2]).all())


def test_add_rmsnorm_special_rows(ops):
    """Zero rows (with and without eps), infinities and NaN stay in their row; large values do not overflow 32 bits where their squares' mean fits."""
    x = rnd((6, 256), torch.float32, 7)
    w = torch.ones(256)
    x[1] = 0
    x[2, 5] = math.inf
    x[3, 9] = math.nan
    x[4] *= 1e17
    total, y = ops.add_rmsnorm(x.cuda(), w.cuda(), torch.zeros_like(x).cuda(), eps=1e-6)
    assert bool((y[1] == 0).all())
    assert bool(y[3].isnan().all()) and bool(y[2, 5].isnan())
    for i in (0, 4, 5):
        assert bool(y[i].isfinite().all())
    for quant in ("int8", "e4m3"):
        _, q, s = ops.add_rmsnorm(x.cuda(), w.cuda(), None, eps=1e-6, quant=quant, group=32)
        v = q.float().reshape(6, 8, 32) * s[..., None]
        assert bool((v[1] == 0).all()) and bool((s[1] == 0).all()) and bool(v[3].isnan().all())
        assert bool(v[0].isfinite().all()) and bool(v[4].isfinite().all())
    ops.sync()


def test_add_rmsnorm_in_place(pkg, ops):
    """The C entry point may put the sum over x or over the residual, whatever kernel the length takes."""
    L, p = ops._L, lambda t: t.data_ptr()  # noqa: E731
    for cols in (256, 250, 5, 8, 9, 1023, 1027, 2047, 4099, 8191, 32763, 33001):
        for quant in (2, 3):                                    # bf16 out, int8 out
            x, r, w = rnd((5, cols), torch.bfloat16, 8).cuda(), rnd((5, cols), torch.bfloat16, 9).cuda(), rnd((cols,), torch.bfloat16, 10).cuda()
            want = ops.add_rmsnorm(x, w, r, eps=1e-5, quant=None if quant == 2 else "int8")
            for into in (0, 1):
                a, b = x.clone(), r.clone()
                y = torch.empty((5, cols), dtype=torch.bfloat16 if quant == 2 else torch.int8, device="cuda")
                s = torch.empty((5, 1), device="cuda")
                rc = L.hipvoc_add_rmsnorm(ops._h, p(a), cols, p(b), cols, p(w), p((a, b)[into]), cols, p(y), cols, None if quant == 2 else p(s), 2, quant, 0, 1e-5,
                                          5, cols, ops.stream)
                assert rc == 0
                assert torch.equal((a, b)[into], want[0]) and torch.equal(y, want[1])
    ops.sync()


@pytest.mark.parametrize("cols", [1, 7, 8, 9, 15, 63, 513, 1025, 2051, 4097, 8195, 32761])
@pytest.mark.parametrize("quant", [None, "int8"])
def test_add_rmsnorm_writes_its_rows_alone(ops, cols, quant):
    """Odd rows inside wider ones, at odd places: what lies between and behind them is left as it was."""
    L, p, rows, wide = ops._L, lambda t: t.data_ptr(), 3, cols + 5  # noqa: E731
    x, r, w = [rnd((n, cols), torch.bfloat16, 30 + n).cuda() for n in (rows, rows, 1)]
    w = w[0].contiguous()
    want = ops.add_rmsnorm(x, w, r, eps=1e-5, quant=quant)
    out = torch.bfloat16 if quant is None else torch.int8
    sums, y = torch.full((rows * wide + 9,), 7.0, dtype=torch.bfloat16, device="cuda"), torch.full((rows * wide + 9,), 7, dtype=out, device="cuda")
    s = torch.empty((rows, 1), device="cuda")
    rc = L.hipvoc_add_rmsnorm(ops._h, p(x), cols, p(r), cols, p(w), p(sums[3:]), wide, p(y[5:]), wide, None if quant is None else p(s), 2, 2 if quant is None else 3, 0,
                              1e-5, rows, cols, ops.stream)
    assert rc == 0
    ops.sync()
    for flat, at, ref in ((sums, 3, want[0]), (y, 5, want[1])):
        keep = torch.full((rows * wide + 9,), 7, dtype=flat.dtype, device="cuda")
        keep[at:at + rows * wide].view(rows, wide)[:, :cols] = ref
        assert torch.equal(flat, keep)


# ---------------------------------------------------------------------------------------------------------------------
# 4-bit products
def q4_weights(n, k, group, mins, seed):
    g = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand((n, k // group), generator=g) * 0.1 - 0.03).to(torch.float16)      # negative ones among them
    least = (torch.randn((n, k // group), generator=g) * 0.3).to(torch.float16) if mins else None
    c = torch.stack((codes & 15, codes >> 4), -1).reshape(n, k).double()
    s = scales.double().repeat_interleave(group, 1)
    w = s * (c - 8) if least is None else s * c + least.double().repeat_interleave(group, 1)
    return codes, scales, least, w, s.abs()


def check_q4(ops, n, k, group, mins, x, x_scale=None, dtype=None, seed=0):
    codes, scales, least, w, s = q4_weights(n, k, group, mins, seed)
    cu = lambda t: None if t is None else t.cuda()  # noqa: E731
    y = ops.q4_matvec(cu(codes), cu(scales), x.cuda() if not x.is_cuda else x, mins=cu(least), x_scale=cu(x_scale), dtype=dtype)
    ops.sync()
    xv = x.cpu().double()
    if x_scale is not None:
        xv = xv * (x_scale.double() if x_scale.shape[1] == 1 else x_scale.double().repeat_interleave(group, 1))
    ref = xv @ w.t()
    # a weight may be carried as code + 16 with 24 (or 16 and the least value) taken off again: no product has a factor over 55 scales
    mag = xv.abs() @ (55 * s).t() + (xv.abs() @ least.double().abs().repeat_interleave(group, 1).t() if mins else 0)
    bound = mag * ((k + 16) * U32) + u(y.dtype) * ref.abs() + 2.0 ** -25 * (y.dtype == torch.float16)
    d = (y.cpu().double() - ref).abs()
    assert y.shape == ref.shape and bool((d <= bound * (1 + u(y.dtype))).all()), float((d / bound).max())
    return y


@pytest.mark.parametrize("act", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("m,n,mult", [(1, 1, 1), (1, 17, 3), (2, 33, 5), (3, 16, 8), (5, 100, 17), (16, 65, 9), (17, 31, 2), (40, 48, 4)])
def test_q4_matvec(ops, act, group, mins, m, n, mult):
    k = group * mult
    check_q4(ops, n, k, group, mins, rnd((m, k), ACT[act], m * 7 + n, 2.0), seed=n + mult)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("mins", [False, True])
@pytest.mark.parametrize("m,n,mult,per_row", [(1, 1, 1, False), (1, 40, 3, True), (4, 33, 9, False), (16, 64, 16, False), (19, 17, 5, True)])
def test_q4_matvec_int8_rows(ops, dtype, group, mins, m, n, mult, per_row):
    k = group * mult
    g = torch.Generator().manual_seed(m + n)
    x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    xs = torch.rand((m, 1 if per_row else mult), generator=g) * 0.02
    check_q4(ops, n, k, group, mins, x, xs, ACT[dtype], seed=mult)


@pytest.mark.parametrize("act,m,n,k", [("bf16", 1, 2048, 1024), ("bf16", 4, 1000, 4096), ("f32", 2, 515, 2048), ("f16", 16, 4100, 1536)])
def test_q4_matvec_larger(ops, act, m, n, k):
    check_q4(ops, n, k, 64, True, rnd((m, k), ACT[act], 2), seed=3)
    check_q4(ops, n, k, 32, False, rnd((m, k), ACT[act], 2), seed=4)


# more weight rows than a tile per CU: other kernels over 4096, 8192 and 16384 of them (counted for every 16 rows of x) and from 65536
@pytest.mark.parametrize("act,n,group,mult,mins,m", [
    ("bf16", 4097, 64, 9, True, 3), ("f16", 8190, 32, 131, False, 1), ("f32", 5003, 128, 3, True, 16), ("int8", 8192, 32, 35, True, 5),
    ("bf16", 8193, 32, 260, False, 2), ("f16", 16384, 64, 19, True, 16), ("f32", 9001, 32, 130, True, 2), ("int8", 12345, 64, 21, False, 9),
    ("bf16", 2050, 64, 17, True, 40), ("f16", 300, 128, 40, False, 900), ("int8", 1000, 32, 33, True, 300), ("f32", 2049, 32, 17, False, 70),
    ("bf16", 16384, 64, 5, True, 3), ("f16", 16390, 32, 33, False, 17), ("bf16", 65541, 128, 3, True, 1), ("f16", 65536, 64, 18, False, 16),
    ("bf16", 65537, 32, 40, True, 2), ("bf16", 16385, 32, 131, True, 5), ("f16", 65540, 32, 128, True, 2), ("bf16", 65536, 32, 123, False, 1),
    ("f16", 65536, 32, 125, False, 33), ("bf16", 16384, 32, 1, True, 1), ("f32", 8192, 64, 9, True, 2), ("f32", 8199, 32, 130, False, 1),
    ("f32", 32769, 64, 5, False, 17), ("f32", 32768, 32, 33, True, 3), ("f32", 32780, 32, 140, True, 1), ("int8", 16399, 64, 5, False, 3),
    ("int8", 16384, 32, 132, True, 18), ("int8", 65536, 32, 127, True, 2), ("int8", 65551, 128, 9, False, 1), ("int8", 100, 32, 300, True, 4),
    ("bf16", 100, 32, 300, True, 4), ("f32", 70, 32, 257, False, 17)])
def test_q4_matvec_many_weight_rows(ops, act, n, group, mult, mins, m):
    """Checked against 64 bits for rows at both ends and a thousand in between; K in whole slabs of 128 columns and not, over 128 groups."""
    k = group * mult
    g = torch.Generator().manual_seed(n + mult)
    scale = None
    if act == "int8":
        x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
        scale = torch.rand((m, mult if mult % 2 else 1), generator=g) * 0.02
    else:
        x = rnd((m, k), ACT[act], m + n, 2.0)
    codes = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scales = (torch.rand((n, mult), generator=g) * 0.1 - 0.03).to(torch.float16)
    least = (torch.randn((n, mult), generator=g) * 0.3).to(torch.float16) if mins else None
    y = ops.q4_matvec(codes.cuda(), scales.cuda(), x.cuda(), mins=None if least is None else least.cuda(), x_scale=None if scale is None else scale.cuda())
    ops.sync()
    pick = torch.unique(torch.cat([torch.arange(min(n, 80)), torch.arange(max(0, n - 300), n), torch.randint(0, n, (1000,), generator=g)]))
    c = torch.stack((codes[pick] & 15, codes[pick] >> 4), -1).reshape(len(pick), k).double()
    s = scales[pick].double().repeat_interleave(group, 1)
    low = least[pick].double().repeat_interleave(group, 1) if mins else 0 * s
    w = s * c + low if mins else s * (c - 8)
    xv = x.double()
    if scale is not None:
        xv = xv * (scale.double().repeat_interleave(group, 1) if scale.shape[1] > 1 else scale.double())
    ref = xv @ w.t()
    mag = xv.abs() @ (55 * s.abs() + low.abs()).t()                                       # as in check_q4
    bound = mag * ((k + 16) * U32) + u(y.dtype) * ref.abs() + 2.0 ** -25 * (y.dtype == torch.float16)
    d = (y.cpu()[:, pick].double() - ref).abs()
    assert y.shape == (m, n) and bool((d <= bound * (1 + u(y.dtype))).all()), float((d / bound).max())


def test_q4_matvec_wide_captured_first(ops):
    """The kernel that asks for more than the default of shared memory, first called under capture."""
    n, k = 65536, 256
    codes, scales, _, _, _ = q4_weights(n, k, 128, False, 1)
    codes, scales = codes.cuda(), scales.cuda()
    x = torch.zeros((2, k), dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.q4_matvec(codes, scales, x)
    for rep in range(3):
        x.copy_(rnd((2, k), torch.float16, rep))
        want = ops.q4_matvec(codes, scales, x)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want) and bool(y.any())


def test_q4_matvec_strides_extremes_and_repeat(ops):
    """Rows inside a wider tensor; codes 0 and 15 throughout; large and small activations; the same bits every time."""
    wide = rnd((5, 512), torch.bfloat16, 5).cuda()
    check_q4(ops, 37, 256, 64, False, wide[:, 128:384])
    k, n, group = 256, 20, 32
    for byte in (0x00, 0xff, 0x0f, 0xf0):
        codes = torch.full((n, k // 2), byte, dtype=torch.uint8, device="cuda")
        scales = torch.ones((n, k // group), dtype=torch.float16, device="cuda")
        for act, size in (("f32", 1e30), ("bf16", 1e30), ("f16", 1.0), ("f32", 1e-30), ("bf16", 1e-30)):
            x = (rnd((3, k), torch.float32, 6) * size).to(ACT[act])
            w = torch.tensor([(byte & 15) - 8, (byte >> 4) - 8], dtype=torch.float64).repeat(k // 2)
            y = ops.q4_matvec(codes, scales, x.cuda())
            ref = (x.double() * w).sum(-1, keepdim=True).expand(3, n)
            mag = (x.double().abs() * 55).sum(-1, keepdim=True)
            assert bool(((y.cpu().double() - ref).abs() <= mag * (k + 16) * U32 + u(ACT[act]) * ref.abs() * 1.01 + 2.0 ** -25 * (act == "f16")).all()), (byte, act, size)
    x = rnd((7, 1024), torch.float16, 7)
    a = check_q4(ops, 333, 1024, 32, True, x)
    b = check_q4(ops, 333, 1024, 32, True, x)
    assert torch.equal(a, b)
    one = check_q4(ops, 333, 1024, 32, True, x[:1])
    assert torch.equal(one[0], a[0])                             # a row's result does not depend on its neighbours
    bad = x.clone()
    bad[2, 5] = math.nan
    codes, scales, least, _, _ = q4_weights(333, 1024, 32, True, 0)
    y = ops.q4_matvec(codes.cuda(), scales.cuda(), bad.cuda(), mins=least.cuda())
    ops.sync()
    assert bool(y[2].isnan().all()) and torch.equal(y[:2], a[:2]) and torch.equal(y[3:], a[3:])
    assert ops.q4_matvec(codes.cuda(), scales.cuda(), x[:0].cuda(), mins=least.cuda()).shape == (0, 333)


# ---------------------------------------------------------------------------------------------------------------------
# streams, graphs, refusals, the operators together
class Layer:
    """One decoder layer's token step: norm -> q, k, v (4 bits) -> cache -> attention -> out projection -> norm -> feed-forward."""

    def __init__(self, hidden=256, heads=8, kv=2, hd=64, ff=512, seed=0):
        self.heads, self.kv, self.hd, self.group = heads, kv, hd, 32
        self.w = {name: q4_weights(n, k, 32, name == "down", seed + i) for i, (name, n, k) in enumerate(
            [("qkv", (heads + 2 * kv) * hd, hidden), ("o", hidden, heads * hd), ("up", ff, hidden), ("down", hidden, ff)])}
        self.dev = {name: [None if t is None else t.cuda() for t in w[:3]] for name, w in self.w.items()}
        self.norm = [(1 + 0.1 * rnd((hidden,), torch.float32, seed + 50 + i)).to(torch.bfloat16) for i in range(2)]
        self.gnorm = [n.cuda() for n in self.norm]

    def project(self, ops, name, x, x_scale=None):
        codes, scales, mins = self.dev[name]
        return ops.q4_matvec(codes, scales, x, mins=mins, x_scale=x_scale, dtype=torch.bfloat16)

    def step(self, ops, x, res, cache, table, lens, cu, first, max_len, keep=None):
        keep = {} if keep is None else keep
        h, c, s = ops.add_rmsnorm(x, self.gnorm[0], res, eps=1e-5, quant="int8", group=32)
        qkv = self.project(ops, "qkv", c, s).reshape(x.shape[0], self.heads + 2 * self.kv, self.hd)
        q, k, v = qkv[:, :self.heads], qkv[:, self.heads:self.heads + self.kv], qkv[:, self.heads + self.kv:]
        ops.kv_write(cache, k, v, table, cu, first)
        a = ops.attention(q, cache, table, lens, max_len=max_len, window=0)
        o = self.project(ops, "o", a.reshape(x.shape[0], -1))
        h2, c2, s2 = ops.add_rmsnorm(o, self.gnorm[1], h, eps=1e-5, quant="int8", group=32)
        f = torch.nn.functional.silu(self.project(ops, "up", c2, s2))
        d = self.project(ops, "down", f)
        keep.update(h=h, c=c, s=s, qkv=qkv, a=a, o=o, h2=h2, c2=c2, s2=s2, f=f, d=d)
        return d, h2


@pytest.mark.parametrize("store", ["same", "int8", "e4m3"])
def test_a_layer_step_by_step(ops, store):
    """Several tokens through one layer, every stage against 64 bits on the stage's own inputs; attention over what the steps wrote."""
    lay, B, page, steps = Layer(), 3, 8, 20
    past = [0, 7, 29]
    P = Paged(ops, past, lay.kv, lay.hd, page, "bf16", store, seed=3, extra_pages=24, width=8)
    used = set(P.table[P.table >= 0].tolist())
    free = iter([p for p in range(P.cache.n_pages) if p not in used])
    P.table = torch.tensor([[p if p >= 0 else next(free) for p in row] for row in P.table.tolist()], dtype=torch.int32, device="cuda")
    x, res = rnd((B, 256), torch.bfloat16, 1).cuda(), rnd((B, 256), torch.bfloat16, 2).cuda()
    for t in range(steps):
        P.lens = [p + t + 1 for p in past]
        P.lens_dev = ints(P.lens)
        keep = {}
        d, h2 = lay.step(ops, x, res, P.cache, P.table, P.lens_dev, ints([0, 1, 2, 3]), ints([n - 1 for n in P.lens]), 64, keep)
        ops.sync()
        kk = {n: v.cpu() for n, v in keep.items()}
        # the products, on the codes that went in
        for name, xin, sc, y in (("qkv", kk["c"], kk["s"], kk["qkv"].reshape(B, -1)), ("o", kk["a"].reshape(B, -1), None, kk["o"]),
                                 ("up", kk["c2"], kk["s2"], None), ("down", kk["f"], None, kk["d"])):
            if y is None:
                continue
            _, _, least, w, s = lay.w[name]
            xv = xin.double() if sc is None else xin.double() * sc.double().repeat_interleave(32, 1)
            ref = xv @ w.t()
            mag = xv.abs() @ (55 * s).t() + (xv.abs() @ least.double().abs().repeat_interleave(32, 1).t() if least is not None else 0)
            assert bool(((y.double() - ref).abs() <= 1.01 * (mag * (xv.shape[1] + 16) * U32 + u(torch.bfloat16) * ref.abs())).all()), name
        # what the step wrote is what attention sees
        new = kk["qkv"][:, lay.heads:]
        for b in range(B):
            for mine, rows in ((P.k, new[b, :lay.kv]), (P.v, new[b, lay.kv:])):
                if store == "same":
                    value = rows.double()
                else:
                    c, sc = encode(rows, store)
                    value = c.double() * sc.double()[..., None]
                mine[b] = torch.cat([mine[b], value[None]])
        ro, _, bo, _ = attention_ref(P, kk["qkv"][:, :lay.heads], 1 / 8, 0)
        assert bool(((kk["a"].double() - ro).abs() <= bo).all())
        x, res = d, h2


def test_a_captured_step_replays_like_the_eager_one(ops):
    """The step under graph capture: replayed several times with new inputs, eager work between the replays, two graphs in turn."""
    lay, B, page = Layer(seed=7), 4, 16
    P = Paged(ops, [3, 500, 0, 2100], lay.kv, lay.hd, page, "bf16", "int8", seed=5)
    P2 = Paged(ops, [900, 5, 33, 1], lay.kv, lay.hd, page, "bf16", "int8", seed=6)
    jobs = []
    for Q in (P, P2):
        pool = list(range(Q.cache.n_pages))
        used = set(Q.table[Q.table >= 0].tolist())
        free = [p for p in pool if p not in used]
        t = Q.table.clone()
        for b, n in enumerate(Q.lens):
            if n % page == 0:                                   # the new token opens a page (there are three to spare)
                t2 = torch.full((4, Q.width + 1), -7, dtype=torch.int32)
                t2[:, :Q.width] = t.cpu()[:, :Q.width]
                t2[b, n // page] = free.pop()
                t = t2.cuda()
        Q.table = t
        lens = ints([n + 1 for n in Q.lens])
        first = ints(Q.lens)
        x, res, cu = torch.zeros((B, 256), dtype=torch.bfloat16, device="cuda"), torch.zeros((B, 256), dtype=torch.bfloat16, device="cuda"), ints([0, 1, 2, 3, 4])
        args = (x, res, Q.cache, Q.table, lens, cu, first, max(Q.lens) + 1)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lay.step(ops, *args)
        torch.cuda.current_stream().wait_stream(side)
        ops.sync()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = lay.step(ops, *args)
        jobs.append((g, args, out))
    for rep in range(4):
        want = []
        for i, (g, args, out) in enumerate(jobs):
            args[0].copy_(rnd((B, 256), torch.bfloat16, 100 + 10 * rep + i))
            args[1].copy_(rnd((B, 256), torch.bfloat16, 200 + 10 * rep + i))
            want.append([t.clone() for t in lay.step(ops, *args)])
        torch.cuda.synchronize()
        for g, _, _ in jobs:
            g.replay()
        torch.cuda.synchronize()
        for (g, _, out), w in zip(jobs, want):
            assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1]), rep
        (torch.ones(1000, device="cuda") * rep).sum().item()
    # both at once, on two streams: they share nothing
    s = [torch.cuda.Stream(), torch.cuda.Stream()]
    for (g, _, _), st in zip(jobs, s):
        with torch.cuda.stream(st):
            for _ in range(5):
                g.replay()
    torch.cuda.synchronize()
    for (g, _, out), w in zip(jobs, want):
        assert torch.equal(out[0], w[0]) and torch.equal(out[1], w[1])
    ops.sync()


def test_calls_follow_the_current_stream(ops):
    """Work on a side stream sees what that stream wrote before, and two streams with one handle do not disturb each other."""
    P = Paged(ops, [700, 1500], 2, 64, 16, "bf16", seed=21)
    q = rnd((2, 8, 64), torch.bfloat16, 3).cuda()
    want = ops.attention(q, P.cache, P.table, P.lens_dev)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(30):
        with torch.cuda.stream(streams[i % 3]):
            late = torch.zeros_like(q)
            late += q                                            # on this stream, just before the call
            outs.append(ops.attention(late, P.cache, P.table, P.lens_dev))
    torch.cuda.synchronize()
    for o in outs:
        assert torch.equal(o, want)


def test_current_device_and_handle_kinds(pkg, ops, synth, tmp_path):
    assert torch.cuda.current_device() == 0
    o = pkg.HipOps.open(0)
    L = o._L
    assert L.hipvoc_decode(o._h, None, 0, None, 0, None) == -1 and b"operator handle" in L.hipvoc_last_error(o._h)
    assert pkg.encoder._lib().hipvoc_enc_n_codebooks(o._h) < 0
    assert L.hipvoc_sync(o._h) == 0
    o.close()
    with pytest.raises(pkg.HipVocError):
        o.sync()
    with pytest.raises(pkg.HipVocError):
        pkg.HipOps.open(99)
    path = str(tmp_path / "w.safetensors")
    synth.save_safetensors(path, synth.make_weights(synth.ODD, 0), synth.ODD.metadata())
    voc = pkg.HipVocoder.load(path, unit_frames=4)
    assert L.hipvoc_ops_sync(voc._h, None) == -1 and b"no operator handle" in L.hipvoc_last_error(voc._h)
    voc.close()


def test_refusals(pkg, ops):
    """Each is refused before a launch, with a text; the handle keeps working."""
    P = Paged(ops, [9, 12], 2, 64, 8, "bf16", seed=1)
    q = rnd((2, 4, 64), torch.bfloat16, 1).cuda()
    x = rnd((2, 64), torch.bfloat16, 1).cuda()
    w = rnd((64,), torch.bfloat16, 1).cuda()
    codes, scales, least, _, _ = [t.cuda() if isinstance(t, torch.Tensor) else t for t in q4_weights(8, 64, 32, True, 0)]
    new = rnd((2, 2, 64), torch.bfloat16, 1).cuda()
    cu, first = ints([0, 1, 2]), ints([9, 12])
    bad = [
        lambda: ops.attention(q[:, :3], P.cache, P.table, P.lens_dev),
        lambda: ops.attention(q.float(), P.cache, P.table, P.lens_dev),
        lambda: ops.attention(q.cpu(), P.cache, P.table, P.lens_dev),
        lambda: ops.attention(q[..., :32], P.cache, P.table, P.lens_dev),
        lambda: ops.attention(q, P.cache, P.table.long(), P.lens_dev),
        lambda: ops.attention(q, P.cache, P.table[:1], P.lens_dev),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev.long()),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev, max_len=17),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev, max_len=2 ** 32 + 5),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev, window=-1),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev, window=2 ** 33),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev, scale=math.nan),
        lambda: ops.attention(q, P.cache, P.table, P.lens_dev, out=q[:1]),
        lambda: ops.kv_write(P.cache, new[:, :1], new[:, :1], P.table, cu, first),
        lambda: ops.kv_write(P.cache, new.half(), new.half(), P.table, cu, first),
        lambda: ops.kv_write(P.cache, new, new, P.table, cu[:2], first),
        lambda: ops.kv_write(P.cache, new, new, P.table, cu.float(), first),
        lambda: ops.kv_write(P.cache, new, new[:1], P.table, cu, first),
        lambda: ops.kv_read(P.cache, P.table, cu, first, 2, dtype=torch.float32),
        lambda: ops.kv_read(P.cache, P.table, cu, first, -1),
        lambda: ops.kv_read(P.cache, P.table, cu, first, 2 ** 40, out=(new, new)),
        lambda: ops.kv_read(P.cache, P.table, cu, first, 3, out=(new, new)),
        lambda: ops.add_rmsnorm(x, w.float()),
        lambda: ops.add_rmsnorm(x, w[:32]),
        lambda: ops.add_rmsnorm(x, w, x[:1]),
        lambda: ops.add_rmsnorm(x, w, quant="int4"),
        lambda: ops.add_rmsnorm(x, w, quant="int8", group=48),
        lambda: ops.add_rmsnorm(x, w, group=32),
        lambda: ops.add_rmsnorm(x, w, eps=-1.0),
        lambda: ops.add_rmsnorm(x, w, eps=math.inf),
        lambda: ops.add_rmsnorm(x.t(), w[:2]),
        lambda: ops.add_rmsnorm(x.int(), w),
        lambda: ops.q4_matvec(codes, scales, x[:, :32]),
        lambda: ops.q4_matvec(codes, scales.float(), x),
        lambda: ops.q4_matvec(codes, scales, x, mins=least[:4]),
        lambda: ops.q4_matvec(codes, scales, x.to(torch.int8)),
        lambda: ops.q4_matvec(codes, scales, x, x_scale=torch.ones((2, 2), device="cuda")),
        lambda: ops.q4_matvec(codes, scales, x, dtype=torch.float32),
        lambda: ops.q4_matvec(codes, scales, x.to(torch.int8), x_scale=torch.ones((2, 3), device="cuda")),
        lambda: ops.q4_matvec(codes.int(), scales, x),
        lambda: ops.q4_matvec(codes, torch.ones((8, 4), dtype=torch.float16, device="cuda"), x),      # groups of 16
        lambda: ops.q4_matvec(codes[:, 1:], scales, x),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(pkg.HipVocError) as e:
            f()
        assert e.value.code == -1, (i, str(e.value))
    P.lens_dev = ints([9, 12])
    check_attention(ops, P, q)


def test_refusals_of_shapes(pkg, ops):
    """What the C side cannot see in a tensor, or would have to divide by."""
    P = Paged(ops, [9], 8, 64, 8, "bf16")
    bf = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    for bad in [lambda: ops.attention(bf(1, 4, 64), P.cache, P.table, P.lens_dev), lambda: ops.attention(bf(1, 12, 64), P.cache, P.table, P.lens_dev),
                lambda: ops.attention(bf(64), P.cache, P.table, P.lens_dev), lambda: ops.attention(bf(1, 0, 64), P.cache, P.table, P.lens_dev),
                lambda: ops.attention(None, P.cache, P.table, P.lens_dev), lambda: ops.attention(bf(1, 8, 64), None, P.table, P.lens_dev),
                lambda: ops.attention(bf(1, 8, 64), P.cache, P.table, P.lens_dev, max_len=1 << 31), lambda: ops.attention(bf(1, 8, 64), P.cache, P.table, P.lens_dev, window=-1),
                lambda: ops.attention(bf(1, 8, 64), P.cache, P.table, P.lens_dev.long()), lambda: ops.attention(bf(1, 8, 64), P.cache, P.table.cpu(), P.lens_dev),
                lambda: ops.attention(bf(1, 8, 64).to_sparse(), P.cache, P.table, P.lens_dev), lambda: ops.attention(bf(1, 8, 64), P.cache, P.table, P.lens_dev, out=bf(2, 8, 64)),
                lambda: ops.kv_read(P.cache, P.table, ints([0, 1]), ints([0]), 1, out=[bf(1, 8, 64)] * 2), lambda: ops.kv_read(P.cache, P.table, ints([0, 1]), ints([0]), -1),
                lambda: ops.kv_read(P.cache, P.table, ints([0, 1]), ints([0]), 1, dtype="bf16"), lambda: ops.kv_read(P.cache, P.table, ints([0, 1]), ints([0]), 1, dtype=torch.int32),
                lambda: ops.add_rmsnorm(bf(2, 8), bf(8), quant="int4"), lambda: ops.add_rmsnorm(bf(2, 8), bf(8), quant="int8", group=-32), lambda: ops.add_rmsnorm(bf(2, 8), bf(9)),
                lambda: ops.add_rmsnorm(bf(1, 8).expand(1 << 22, 8).contiguous(), bf(8)), lambda: ops.add_rmsnorm(bf(1, 8).expand(4, 8), bf(8))]:
        with pytest.raises(pkg.HipVocError) as e:
            bad()
        assert e.value.code == -1 and len(str(e.value)) > 5
    ops.sync()


def test_a_closed_handle_refuses(pkg):
    o = pkg.HipOps.open(0)
    o.close()
    for call in (lambda: o.add_rmsnorm(torch.zeros((1, 8), device="cuda"), torch.zeros(8, device="cuda")), o.sync):
        with pytest.raises(pkg.HipVocError):
            call()
    o.close()


def test_outputs_keep_to_their_calls(ops):
    """Results are tensors of their own: no call writes into what an earlier one gave, and what they hold is freed with them."""
    x, w = rnd((64, 256), torch.float32, 1).cuda(), torch.ones(256, device="cuda")
    first = ops.add_rmsnorm(x, w)[1]
    kept = first.clone()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for i in range(200):
        ops.add_rmsnorm(x + i, w, x)
    torch.cuda.synchronize()
    assert torch.equal(first, kept) and torch.cuda.memory_allocated() == before


def test_calls_from_several_threads(pkg, ops):
    """One handle, four threads with a stream each: sound calls give what they give alone, refused ones their code and a text."""
    import threading
    w = (1 + 0.1 * rnd((512,), torch.float32, 1)).cuda()
    xs = [rnd((33, 512), torch.float32, 10 + i).cuda() for i in range(4)]
    want = [ops.add_rmsnorm(x, w)[1].clone() for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(60):
                    got = ops.add_rmsnorm(xs[i], w)[1]
                    try:
                        ops.add_rmsnorm(xs[i], w, eps=-1.0)
                        wrong.append("not refused")
                    except pkg.HipVocError as e:
                        if e.code != -1 or "eps" not in str(e):
                            wrong.append(str(e))
                    ops.sync()
                    if not torch.equal(got, want[i]):
                        wrong.append("differs")
        except Exception as e:  # noqa: BLE001
            wrong.append(repr(e))
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong, wrong[:3]
