"""The cache held in 8 bits: its write against the definition bit by bit, attention over it against 64 bits."""

import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(np.asarray(x, dtype=np.int32), device=DEV)


class Step:
    """A step of requests (tokens brought, keys afterwards) over a pool of pages in random order."""

    def __init__(self, lengths, nh, nkv, hd, ps, dtype, seed=0, q_stride=None):
        self.lengths, self.nh, self.nkv, self.hd, self.ps, self.dtype = lengths, nh, nkv, hd, ps, dtype
        g = torch.Generator().manual_seed(seed)
        need = [-(-kv // ps) for _, kv in lengths]
        self.pool = sum(need) + 3
        perm = torch.randperm(self.pool, generator=g).tolist()
        self.first = np.concatenate([[0], np.cumsum(need)]).astype(int)
        self.ids = perm[: int(self.first[-1])]
        self.starts = np.concatenate([[0], np.cumsum([q for q, _ in lengths])]).astype(int)
        self.T = int(self.starts[-1])
        self.seq = np.concatenate([np.full(q, s) for s, (q, _) in enumerate(lengths)] or [[]]).astype(int)
        self.pos = np.concatenate([np.arange(kv - q, kv) for q, kv in lengths] or [[]]).astype(int)
        shape = (self.pool, nkv, ps, hd)
        self.kc = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).to(DEV)
        self.vc = torch.randint(-127, 128, shape, generator=g, dtype=torch.int8).to(DEV)
        self.ks = (torch.rand(self.pool, nkv, generator=g) * 0.03 + 1e-3).to(DEV)
        self.vs = (torch.exp(2 * torch.randn(self.pool, nkv, generator=g)) * 0.01).to(DEV)
        self.rows = torch.randn(self.T, (nh + 2 * nkv) * hd, generator=g).to(dtype).to(DEV)
        buf = torch.randn(self.T, q_stride or nh * hd, generator=g).to(dtype).to(DEV)
        self.q = buf[:, : nh * hd]
        self.status = torch.zeros(1, dtype=torch.int32, device=DEV)

    def write(self, inv_freq=None, rot=0, write_cache=True, rows=None):
        from tokasaurus_b200.kernels import int8

        int8.rope_kv8_write(self.rows if rows is None else rows, i32(self.pos), i32(self.seq), i32(self.first), i32(self.ids), inv_freq,
                            self.kc, self.vc, self.ks, self.vs, self.nh, self.nkv, self.hd, rot, self.ps, write_cache, self.status)

    def attend(self, window=None, scale=None, ids=None):
        from tokasaurus_b200.kernels import int8

        out = torch.full((self.T, self.nh * self.hd), float("nan"), dtype=self.dtype, device=DEV)
        q_len, kv_len = [q for q, _ in self.lengths], [kv for _, kv in self.lengths]
        int8.attn_kv8(self.q, out, self.kc, self.vc, self.ks, self.vs, i32(self.starts[:-1]), i32(q_len), i32(kv_len), i32(self.first),
                      i32(self.ids if ids is None else ids), self.nh, self.nkv, self.hd, self.ps, scale or self.hd**-0.5, window,
                      self.status, max_q_len=max(q_len), max_kv_len=max(kv_len), single_tokens=sum(q == 1 for q in q_len))
        return out

    def check_attention(self, window=None, scale=None, ids=None, rows=None):
        """Against 64 bits on the same codes, with the error that the kernels' roundings can make."""
        out = self.attend(window, scale, ids)
        ids = np.asarray(self.ids if ids is None else ids)
        scale = scale or self.hd**-0.5
        g = self.nh // self.nkv
        low = self.dtype == BF
        for s, (q, kv) in enumerate(self.lengths):
            if q == 0:
                continue
            pages = ids[self.first[s]:self.first[s + 1]]
            at = torch.from_numpy(np.where(pages >= 0, pages, 0)).to(DEV)
            here = torch.from_numpy(np.repeat(pages >= 0, self.ps)[:kv]).to(DEV)
            k = (self.kc[at].double() * self.ks[at].double()[:, :, None, None]).transpose(1, 2).reshape(-1, self.nkv, self.hd)[:kv]
            v = (self.vc[at].double() * self.vs[at].double()[:, :, None, None]).transpose(1, 2).reshape(-1, self.nkv, self.hd)[:kv]
            t0 = int(self.starts[s])
            qq = self.q[t0:t0 + q].double().view(q, self.nkv, g, self.hd)
            sc = torch.einsum("qhgd,khd->hgqk", qq, k) * scale
            mag = torch.einsum("qhgd,khd->hgqk", qq.abs(), k.abs()) * scale
            pos, j = torch.arange(kv - q, kv, device=DEV), torch.arange(kv, device=DEV)
            see = (j <= pos[:, None]) & here
            if window:
                see &= j > pos[:, None] - window
            p = torch.exp(sc - sc.masked_fill(~see, -math.inf).amax(-1, keepdim=True).clamp_min(-1e300)).masked_fill(~see, 0)
            total = p.sum(-1, keepdim=True)
            p = torch.where(total > 0, p / total, 0.0)
            want = torch.einsum("hgqk,khd->qhgd", p, v).reshape(q, -1)
            vmax = (v.abs() * here[:, None, None]).amax((0, 2)).repeat_interleave(g)  # [heads]
            err_s = mag.masked_fill(~see, 0).amax(-1).permute(2, 0, 1).reshape(q, self.nh) * (self.hd * 2.0**-23 + (0 if low else 2.0**-21))
            # weights: the scores' error twice, the exponential, the rounding to what the tensor cores take; the result's rounding
            rel = 2.1 * err_s + 2.0**-20 + (2.0**-10 if low else 2.0**-20)
            bound = (rel * vmax).repeat_interleave(self.hd, 1) + want.abs() * (2.0**-8 if low else 2.0**-23) + 1e-30
            got = out[t0:t0 + q].double()
            far = (got - want).abs() - bound
            assert not got.isnan().any() and (far <= 0).all(), f"request {s}: off by {float(far.max()):.3g} beyond its bound"
        assert int(self.status) == 0
        return out


def plain_write(step, rows, side, cache, scales):
    """The definition in numpy float32, segment by segment; returns the new codes and scales."""
    cache, scales = cache.cpu().numpy().copy(), scales.cpu().numpy().copy()
    x = rows.float().cpu().numpy()[:, (step.nh + side * step.nkv) * step.hd:][:, : step.nkv * step.hd].reshape(-1, step.nkv, step.hd)
    inv = np.float32(1 / 127)
    for s, (q, kv) in enumerate(step.lengths):
        t = int(step.starts[s])
        p = kv - q
        while p < kv:
            n = min(step.ps - p % step.ps, kv - p)
            page = step.ids[step.first[s] + p // step.ps]
            for h in range(step.nkv):
                new = x[t:t + n, h]
                old = np.float32(0) if p % step.ps == 0 else scales[page, h]
                top = np.abs(new).max() * inv
                sc = np.float32(np.nan) if not np.isfinite(new).all() or np.isnan(old) else max(old, top)
                block = cache[page, h].astype(np.float32) * old
                block[p % step.ps: p % step.ps + n] = new
                with np.errstate(all="ignore"):
                    c = np.clip(np.rint(block / sc), -127, 127) if sc > 0 else np.zeros_like(block)
                cache[page, h], scales[page, h] = c.astype(np.int8), sc
            t, p = t + n, p + n
    return cache, scales


MIXES = [
    [(1, 1)], [(1, 16), (1, 17), (1, 15), (1, 300)], [(5, 5)], [(40, 40), (1, 33), (24, 61), (2, 18)], [(100, 131), (3, 3), (1, 2)],
    [(1, 8)] * 70,
]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd,ps", [(4, 2, 16, 16), (3, 1, 32, 8), (32, 8, 64, 16), (8, 8, 128, 16), (4, 2, 80, 5), (2, 1, 256, 64), (2, 2, 48, 1)])
@pytest.mark.parametrize("mix", range(len(MIXES)))
def test_write_as_defined(mix, nh, nkv, hd, ps, dtype):
    st = Step(MIXES[mix], nh, nkv, hd, ps, dtype, seed=mix)
    st.ks[::2] *= 50  # some blocks keep their scale, some have theirs grown
    want = [plain_write(st, st.rows, side, c, s) for side, (c, s) in enumerate(((st.kc, st.ks), (st.vc, st.vs)))]
    before = st.rows.clone()
    for _ in range(2):  # writing the same tokens again changes nothing
        st.write()
        for (wc, ws), c, s in zip(want, (st.kc, st.vc), (st.ks, st.vs)):
            assert np.array_equal(s.cpu().numpy(), ws) and np.array_equal(c.cpu().numpy(), wc)
    assert torch.equal(st.rows, before) and int(st.status) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rot", [16, 64, 24])
def test_write_rotates(rot, dtype):
    """q as ``rope_kv_write`` rotates it, k within half a code of the rotated numbers."""
    from tokasaurus_b200.kernels import int8, ops

    st = Step([(40, 70), (1, 5000), (1, 16), (17, 17)], 8, 2, 64, 16, dtype, seed=5)
    inv = (10000.0 ** (-torch.arange(rot // 2) * 2 / rot)).float().to(DEV)
    ref = st.rows.clone()
    k32 = torch.zeros(st.pool, 2, 16, 64, device=DEV, dtype=dtype)
    v32 = torch.zeros_like(k32)
    ops.rope_kv_write(ref, i32(st.pos), i32(st.seq), i32(st.first), i32(st.ids), inv, k32, v32, 8, 2, 64, rot, 16, True, st.status)
    raw = st.rows.clone()
    st.write(inv, rot)
    assert (st.rows[:, : 8 * 64].double() - ref[:, : 8 * 64].double()).abs().max() <= (2.0**-6 if dtype == BF else 2.0**-18)
    assert torch.equal(st.rows[:, 8 * 64:], raw[:, 8 * 64:])
    k, v = int8.read_kv8(st.kc, st.vc, st.ks, st.vs, i32(np.arange(st.pool)), st.status)
    for s, (q, kv) in enumerate(st.lengths):
        for p in range(kv - q, kv):
            page, slot = st.ids[st.first[s] + p // 16], p % 16
            for got, want, sc in ((k, k32, st.ks), (v, v32, st.vs)):
                w = want[page, :, slot].double()
                off = (got[page, :, slot].double() - w).abs()
                assert (off <= sc[page].double()[:, None] * 0.501 + w.abs() * (2.0**-8 if dtype == BF else 2.0**-20)).all()
    assert int(st.status) == 0


def test_write_of_numbers_that_are_none_and_of_zeros():
    st = Step([(20, 20), (1, 30)], 2, 2, 32, 8, F32)
    rows = st.rows.clone()
    rows[3, 2 * 32 + 5] = float("inf")      # k of head 0, first page
    rows[17, 4 * 32 + 33] = float("nan")    # v of head 1, third page
    rows[8:16, 2 * 32 + 32:2 * 32 + 64] = 0  # k of head 1, second page: all zeros
    want = [plain_write(st, rows, side, c, s) for side, (c, s) in enumerate(((st.kc, st.ks), (st.vc, st.vs)))]
    st.write(rows=rows)
    for (wc, ws), c, s in zip(want, (st.kc, st.vc), (st.ks, st.vs)):
        assert np.array_equal(s.cpu().numpy(), ws, equal_nan=True) and np.array_equal(c.cpu().numpy(), wc)
    assert np.isnan(want[0][1][st.ids[0], 0]) and np.isnan(want[1][1][st.ids[2], 1]) and want[0][1][st.ids[1], 1] == 0


def test_write_skips_padding_and_pages_that_are_none():
    st = Step([(1, 9), (1, 20), (6, 6)], 2, 1, 16, 8, BF)
    kc, vc, ks = st.kc.clone(), st.vc.clone(), st.ks.clone()
    st.write(write_cache=False)
    assert torch.equal(st.kc, kc) and torch.equal(st.ks, ks)
    st.seq[:] = -1
    st.write()
    assert torch.equal(st.kc, kc) and torch.equal(st.vc, vc) and int(st.status) == 0
    st.seq[:] = [0, 1, 2, 2, 2, 2, 2, 2]
    st.ids[int(st.first[1]) + 2] = st.pool + 5
    st.ids[int(st.first[2])] = -1
    st.write()
    assert int(st.status) == 2
    assert torch.equal(st.kc[st.ids[int(st.first[1])]], kc[st.ids[int(st.first[1])]])


def test_read_gives_values_and_zeros_for_no_page():
    from tokasaurus_b200.kernels import int8

    st = Step([(1, 50)], 4, 2, 80, 4, F32)
    pages = [2, 0, -1, 5, 5, st.pool]
    k, v = int8.read_kv8(st.kc, st.vc, st.ks, st.vs, i32(pages), st.status)
    for n, p in enumerate(pages):
        ok = 0 <= p < st.pool
        for got, c, s in ((k, st.kc, st.ks), (v, st.vc, st.vs)):
            want = c[p].float() * s[p][:, None, None] if ok else torch.zeros(2, 4, 80, device=DEV)
            assert torch.equal(got[n], want)
    assert int(st.status) == 2
    assert int8.read_kv8(st.kc, st.vc, st.ks, st.vs, i32([]), st.status)[0].shape == (0, 2, 4, 80)


HEADS = [(32, 8, 64, 16), (32, 8, 128, 16), (24, 8, 128, 16), (3, 1, 32, 8), (4, 2, 16, 16), (8, 8, 80, 16), (12, 1, 64, 32), (20, 1, 96, 16),
         (6, 2, 256, 16), (8, 4, 64, 5), (5, 5, 48, 1), (16, 2, 64, 64), (4, 1, 128, 256), (2, 1, 240, 24)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd,ps", HEADS)
def test_attention_of_single_tokens(nh, nkv, hd, ps, dtype):
    Step([(1, kv) for kv in (1, 2, 15, 16, 17, 63, 64, 65, 200, 511, 1300)], nh, nkv, hd, ps, dtype, seed=hd).check_attention()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("nh,nkv,hd,ps", HEADS)
def test_attention_of_portions(nh, nkv, hd, ps, dtype):
    Step([(2, 2), (1, 77), (40, 40), (130, 197), (3, 500), (1, 1), (65, 400)], nh, nkv, hd, ps, dtype, seed=hd + 1).check_attention()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [1, 7, 16, 50, 64, 300])
@pytest.mark.parametrize("nh,nkv,hd,ps", [(8, 2, 64, 16), (3, 1, 32, 8), (4, 2, 128, 16)])
def test_attention_within_a_window(nh, nkv, hd, ps, window, dtype):
    st = Step([(1, 5), (1, 700), (90, 333), (200, 200), (1, 64), (24, 61)], nh, nkv, hd, ps, dtype, seed=window)
    want = st.check_attention(window)
    # pages behind every token's window were given back
    ids = list(st.ids)
    for s, (q, kv) in enumerate(st.lengths):
        for i in range(max(0, kv - q - window + 1) // ps):
            ids[st.first[s] + i] = -1
    assert torch.equal(st.attend(window, ids=ids), want)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_see_nothing_are_zero(dtype):
    st = Step([(1, 40), (30, 60), (1, 200), (0, 0), (20, 20)], 8, 2, 64, 16, dtype)
    ids = list(st.ids)
    for s in (0, 1):
        for i in range(st.first[s], st.first[s + 1]):
            ids[i] = -1
    ids[st.first[2] + 3] = -1  # a page in the middle is gone
    ids[st.first[4]] = -1      # the first 16 tokens see nothing, the last four each other
    out = st.check_attention(ids=ids)
    assert (out[:31] == 0).all() and (out[32:48] == 0).all() and (out[48:] != 0).any()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[(1, 100), (1, 900)], [(70, 100), (150, 900)]])
def test_what_is_not_seen_may_be_anything(lengths, dtype):
    """Blocks beyond a request's keys, behind the window and on other pages hold NaN scales: no result moves."""
    st = Step(lengths, 8, 2, 64, 16, dtype, seed=3)
    window = 200
    want = st.attend(window)
    live = {st.ids[st.first[s] + i] for s, (q, kv) in enumerate(lengths) for i in range(max(0, kv - q - window + 1) // 16, -(-kv // 16))}
    dead = torch.tensor([p not in live for p in range(st.pool)], device=DEV)
    assert dead.any()
    st.ks[dead], st.vs[dead] = float("nan"), float("inf")
    assert torch.equal(st.attend(window), want)
    # a block that is NaN reaches the tokens that see it, and no others
    st.vs[st.ids[st.first[1] - 1], 0] = float("nan")  # the last block of request 0, kv head 0
    got = st.attend(window)
    q0, kv0 = lengths[0]
    sees = torch.arange(kv0 - q0, kv0, device=DEV) >= (kv0 - 1) // 16 * 16
    head = torch.arange(8 * 64, device=DEV) < 4 * 64
    assert got[:q0][sees][:, head].isnan().all() and torch.equal(got[:q0][~sees], want[:q0][~sees])
    assert torch.equal(got[:q0][:, ~head], want[:q0][:, ~head]) and torch.equal(got[q0:], want[q0:])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lengths", [[(1, 400)], [(33, 400)]])
def test_scales_and_queries_of_every_size(lengths, dtype):
    """Values whose blocks differ by 1e30, queries of 1e-20 and of 1e4, scores so large that one key takes all."""
    st = Step(lengths, 8, 2, 64, 16, dtype, seed=11)
    st.vs *= torch.logspace(-15, 15, st.pool, device=DEV)[torch.randperm(st.pool, device=DEV)][:, None]
    st.check_attention()
    st.vs.fill_(0.01)
    st.q.mul_(1e-20)
    st.check_attention()
    st.q.mul_(1e24)
    st.check_attention(scale=1e-5)
    st.vs.zero_()
    assert (st.attend() == 0).all()


def test_a_long_cache_beyond_32_bit_offsets():
    """Two requests of a pool of 2.4e9 codes a side, on pages whose offsets pass 2^31."""
    from tokasaurus_b200.kernels import int8

    nkv, ps, hd = 8, 64, 256
    pool = 2_400_000_000 // (nkv * ps * hd)
    st = Step([(1, 640), (20, 300)], 16, nkv, hd, ps, BF)
    kc, vc = (torch.zeros(pool, nkv, ps, hd, dtype=torch.int8, device=DEV) for _ in range(2))
    ks, vs = (torch.zeros(pool, nkv, device=DEV) for _ in range(2))
    far = pool - 1 - np.arange(st.pool)
    for dst, src in ((kc, st.kc), (vc, st.vc), (ks, st.ks), (vs, st.vs)):
        dst[torch.from_numpy(far).to(DEV)] = src
    want_out = st.attend()
    st.write()
    want = int8.read_kv8(st.kc, st.vc, st.ks, st.vs, i32(st.ids), st.status)
    st2 = Step([(1, 640), (20, 300)], 16, nkv, hd, ps, BF)
    st2.kc, st2.vc, st2.ks, st2.vs, st2.pool = kc, vc, ks, vs, pool
    st2.ids = [int(far[p]) for p in st2.ids]
    assert torch.equal(st2.attend(), want_out)
    st2.write()
    got = int8.read_kv8(kc, vc, ks, vs, i32(st2.ids), st2.status)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and int(st2.status) == 0


def test_attention_of_strided_queries_and_of_no_tokens():
    st = Step([(1, 90), (33, 50)], 8, 2, 64, 16, BF, q_stride=8 * 64 + 2 * 2 * 64)
    st.check_attention()
    from tokasaurus_b200.kernels import int8

    empty = i32([])
    int8.attn_kv8(st.q[:0], st.q[:0], st.kc, st.vc, st.ks, st.vs, empty, empty, empty, i32([0]), empty, 8, 2, 64, 16, 0.1, None, st.status,
                  max_q_len=0, max_kv_len=0, single_tokens=0)


def test_attention_reports_a_page_beyond_the_pool():
    for lengths in ([(1, 100)], [(20, 100)]):
        st = Step(lengths, 4, 2, 64, 16, BF)
        ids = list(st.ids)
        ids[2] = st.pool + 7
        out = st.attend(ids=ids)
        assert int(st.status) == 2 and not out.isnan().any()
        st.status.zero_()
        ids[2] = -1
        assert torch.equal(st.attend(ids=ids), out) and int(st.status) == 0


def test_same_bits_twice():
    st = Step([(1, 3000)] * 5 + [(200, 900)], 32, 8, 64, 16, BF)
    assert torch.equal(st.attend(), st.attend())


def test_refusals():
    from tokasaurus_b200.kernels import int8
    from tokasaurus_b200.kernels.ops import KernelError

    st = Step([(1, 40), (3, 20)], 4, 2, 64, 16, BF)
    q_len, kv_len, out = i32([1, 3]), i32([40, 20]), torch.empty(4, 256, dtype=BF, device=DEV)

    def attend(**kw):
        a = dict(q=st.q, out=out, kcache=st.kc, vcache=st.vc, k_scale=st.ks, v_scale=st.vs, q_start=i32([0, 1]), q_len=q_len, kv_len=kv_len,
                 page_indptr=i32(st.first), page_ids=i32(st.ids), n_heads=4, n_kv_heads=2, head_dim=64, page_size=16, scale=0.1, window=None,
                 status=st.status, max_q_len=3, max_kv_len=40, single_tokens=1)
        a.update(kw)
        int8.attn_kv8(**a)

    def write(**kw):
        a = dict(qkv=st.rows, positions=i32(st.pos), token_seq=i32(st.seq), page_indptr=i32(st.first), page_ids=i32(st.ids), inv_freq=None,
                 kcache=st.kc, vcache=st.vc, k_scale=st.ks, v_scale=st.vs, n_heads=4, n_kv_heads=2, head_dim=64, rotary_dim=0, page_size=16,
                 write_cache=True, status=st.status)
        a.update(kw)
        int8.rope_kv8_write(**a)

    attend()
    write()
    for call, kw in ((attend, dict(q=st.q.half())), (attend, dict(out=out.float())), (attend, dict(kcache=st.kc.float())),
                     (attend, dict(kcache=st.kc.cpu())), (attend, dict(k_scale=st.ks[:, :1])), (attend, dict(v_scale=st.vs.double())),
                     (attend, dict(n_heads=3)), (attend, dict(page_size=8)), (attend, dict(window=0)), (attend, dict(q_len=q_len.long())),
                     (attend, dict(head_dim=40)), (attend, dict(out=out[:2])), (attend, dict(single_tokens=3)), (attend, dict(q_start=i32([0]))),
                     (attend, dict(vcache=st.vc[1:])), (attend, dict(n_heads=8)), (write, dict(qkv=st.rows[:, :-1])), (write, dict(qkv=st.rows.half())),
                     (write, dict(kcache=st.kc.short())), (write, dict(rotary_dim=64)), (write, dict(rotary_dim=63)), (write, dict(positions=i32([0]))),
                     (write, dict(positions=i32(st.pos).long())), (write, dict(k_scale=st.ks.t())), (write, dict(head_dim=32)),
                     (write, dict(qkv=st.rows.cpu()))):
        with pytest.raises(KernelError):
            call(**kw)
    for bad in (dict(pages=i32([0]).long()), dict(kcache=st.kc[:, :1])):
        a = dict(kcache=st.kc, vcache=st.vc, k_scale=st.ks, v_scale=st.vs, pages=i32([0]), status=st.status)
        a.update(bad)
        with pytest.raises(KernelError):
            int8.read_kv8(**a)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("ps", [5, 64, 256])
def test_write_rotates_into_pages_of_other_sizes(ps, dtype):
    """Portions that fill parts of pages, whole pages and several, with the numbers rotated: codes are those of the numbers that the
    rotation with pages of 16 gives."""
    lengths = [(300, 333), (1, 70), (64, 64), (7, 130)]
    st, ref = Step(lengths, 4, 2, 64, ps, dtype, seed=9), Step(lengths, 4, 2, 64, 16, dtype, seed=9)
    ref.rows = st.rows.clone()
    inv = (10000.0 ** (-torch.arange(32) / 32)).float().to(DEV)
    from tokasaurus_b200.kernels import int8, ops

    k = torch.zeros(st.pool, 2, ps, 64, device=DEV, dtype=dtype)
    v = torch.zeros_like(k)
    plain = st.rows.clone()
    ops.rope_kv_write(plain, i32(st.pos), i32(st.seq), i32(st.first), i32(st.ids), inv, k, v, 4, 2, 64, 64, ps, True, st.status)
    st.write(inv, 64)
    ref.write(inv, 64)
    assert torch.equal(st.rows, ref.rows)  # q does not know of pages
    got = int8.read_kv8(st.kc, st.vc, st.ks, st.vs, i32(np.arange(st.pool)), st.status)
    for s, (q, kv) in enumerate(lengths):
        for p in range(kv - q, kv):
            page, slot = st.ids[st.first[s] + p // ps], p % ps
            for g, want, sc in ((got[0], k, st.ks), (got[1], v, st.vs)):
                w = want[page, :, slot].double()
                # half a code, and half a code again if the block's scale grew later; the rotation's rounding
                grew = 1.0 if (kv - q) % ps else 0.5
                assert ((g[page, :, slot].double() - w).abs() <= sc[page].double()[:, None] * (grew + 0.001) + w.abs() * (2.0**-8 if dtype == BF else 2.0**-20)).all()
    assert int(st.status) == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("q_stride", [8 * 64 + 1, 8 * 64 + 4])
def test_attention_of_rows_on_any_boundary(q_stride, dtype):
    st = Step([(1, 700), (70, 150), (1, 3)], 8, 2, 64, 16, dtype, q_stride=q_stride)
    want = st.check_attention()
    q = st.q
    st.q = q.contiguous()
    assert torch.equal(st.attend(), want)


@pytest.mark.parametrize("hd", [64, 128])
def test_attention_in_a_graph_with_other_lengths(hd):
    """A launch that is replayed: the requests' lengths change in place, up to what the launch was sized for; idle rows bring none."""
    from tokasaurus_b200.kernels import int8

    n = 6
    st = Step([(1, 4000)] * n, 8, 2, hd, 16, BF, seed=2)
    q_len, kv_len = i32([1] * n), i32([4000] * n)
    out = torch.empty(n, 8 * hd, dtype=BF, device=DEV)

    def call():
        int8.attn_kv8(st.q, out, st.kc, st.vc, st.ks, st.vs, i32_starts, q_len, kv_len, first, ids, 8, 2, hd, 16, hd**-0.5, None, st.status,
                      max_q_len=1, max_kv_len=4000, single_tokens=n)

    i32_starts, first, ids = i32(st.starts[:-1]), i32(st.first), i32(st.ids)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
        call()  # (two launches of one step share the graph's memory)
    for lengths in ([4000] * n, [1, 4000, 17, 600, 2000, 3], [5] * n, [3999, 0, 0, 0, 0, 0], [4000] * n):
        q_len.copy_(i32([int(kv > 0) for kv in lengths]))
        kv_len.copy_(i32(lengths))
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        live = [s for s in range(n) if lengths[s] > 0]
        alone = Step([(1, max(kv, 1)) for kv in lengths], 8, 2, hd, 16, BF, seed=2)
        alone.kc, alone.vc, alone.ks, alone.vs, alone.pool = st.kc, st.vc, st.ks, st.vs, st.pool
        alone.q = st.q
        alone.ids = [st.ids[st.first[s] + i] for s in range(n) for i in range(-(-max(lengths[s], 1) // 16))]
        want = alone.check_attention()
        # the same keys in other shares: float32 sums in another order, and the result's rounding
        assert ((out[live].double() - want[live].double()).abs() <= want[live].double().abs() * 2.0**-7 + 2.0**-10 * 127 * st.vs.max().double()).all()
    assert int(st.status) == 0


def test_attention_and_write_on_another_stream():
    st, ref = (Step([(1, 2000)] * 4 + [(50, 90)], 8, 2, 64, 16, BF, seed=4) for _ in range(2))
    ref.write()
    want = ref.attend()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        st.write()
        got = st.attend()
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(st.kc, ref.kc) and torch.equal(st.vs, ref.vs)
