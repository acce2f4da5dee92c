"""Shared-prefix attention over pages against the formula in 64 bits.

Tolerance of an output element, with u the type's half step, s the scores, p the softmax weights
and A = sum p |v|:
  * the weights are rounded to the type before the product with v: u A (fp16 also has an absolute
    half step of 2^-25 below its normal range, each weight relative to a denominator >= 1: 2^-25 sum |v|),
  * the output is rounded: u |o|,
  * a score is a 32-bit sum of hd products, each step off by at most 2^-23 of sum |q k| (tensor
    cores may truncate), then scaled: an error e of a score changes a weight by a factor e^(2e) at most,
    so 4 e A with the denominator's share; the exponential itself adds 2^-21,
  * the sums over positions add 2^-23 per step of 8 positions: n / 8 * 2^-23 A.
"""
import math

import pytest
import torch

from estudiocanciones_b200 import _lib
from estudiocanciones_b200._lib import HMError

pytestmark = pytest.mark.gpu

DEV = "cuda"
H, BF = torch.float16, torch.bfloat16


@pytest.fixture(scope="module", autouse=True)
def _built():
    from estudiocanciones_b200 import build, kernels
    build.build()
    kernels.read_errors(DEV)
    yield
    assert kernels.read_errors(DEV) == 0, "a kernel reported an error bit"


class Case:
    """Sequences in groups on one layer's pool; every slot that no sequence holds is NaN.

    groups: [(plen, [positions held by each sequence])]; a sequence's row 0 .. S - 1 stand at its last S
    positions (below 0: padding rows)."""

    def __init__(self, groups, S=1, Hq=6, Hk=2, hd=128, page=64, dtype=H, seed=0, extra=3, amp=1.0):
        g = torch.Generator().manual_seed(seed)
        self.S, self.Hq, self.Hk, self.hd, self.page, self.dtype = S, Hq, Hk, hd, page, dtype
        lens = [n for _, ns in groups for n in ns]
        B = self.B = len(lens)
        width = max(1, max(-(-max(n, p) // page) for p, ns in groups for n in ns))
        need = sum(p // page + sum(-(-max(0, n) // page) + 1 for n in ns) for p, ns in groups)
        n_pages = need + extra
        order = torch.randperm(n_pages, generator=g).tolist()
        k = torch.full((n_pages, Hk, page, hd), float("nan"), dtype=dtype)
        v = k.clone()
        table = [[-1] * width for _ in range(B)]
        gstart, owner, plen, b = [0], [], [], 0
        for p, ns in groups:
            shared = [order.pop() for _ in range(p // page)]
            kp = torch.randn(p, Hk, hd, generator=g).mul(amp).to(dtype)
            vp = torch.randn(p, Hk, hd, generator=g).to(dtype)
            own = b
            for n in ns:
                if n > max(lens[own], 0):
                    own = b
                held = max(0, -(-n // page))
                pages = [shared[j] if j < len(shared) else order.pop() for j in range(held)]
                table[b][:held] = pages
                kk = torch.cat([kp[:max(n, 0)], torch.randn(max(0, n - p), Hk, hd, generator=g).mul(amp).to(dtype)])
                vv = torch.cat([vp[:max(n, 0)], torch.randn(max(0, n - p), Hk, hd, generator=g).to(dtype)])
                for j, pg in enumerate(pages):
                    m = min(page, n - j * page)
                    if not (j < len(shared) and n < (j + 1) * page):   # a shared page is written by its longest holder
                        k[pg, :, :m] = kk[j * page:j * page + m].transpose(0, 1)
                        v[pg, :, :m] = vv[j * page:j * page + m].transpose(0, 1)
                    else:
                        k[pg] = kp[j * page:(j + 1) * page].transpose(0, 1)
                        v[pg] = vp[j * page:(j + 1) * page].transpose(0, 1)
                b += 1
            owner.append(own)
            plen.append(p if max([0] + ns) >= p else 0)
            gstart.append(b)
        i32 = dict(dtype=torch.int32, device=DEV)
        self.k, self.v = k.to(DEV), v.to(DEV)
        self.q = torch.randn(B * S, Hq * hd, generator=g).mul(1.5 * amp).to(dtype).to(DEV)
        self.table = torch.tensor(table, **i32)
        self.pos = torch.tensor([n - S + s for n in lens for s in range(S)], device=DEV)
        self.gstart, self.owner, self.plen = (torch.tensor(x, **i32) for x in (gstart, owner, plen))
        self.seqs = None

    def run(self, **kw):
        from estudiocanciones_b200 import kernels
        a = dict(gstart=self.gstart, owner=self.owner, plen=self.plen, S=self.S, seqs=self.seqs)
        a.update(kw)
        return kernels.prefix_attn(self.q, self.k, self.v, self.table, self.pos, **a)

    def slots(self, r):
        """(pages, slots) that row r attends to, by the documented rules."""
        b = r // self.S
        row = b if self.seqs is None else int(self.seqs[b])
        n = int(self.pos[r]) + 1
        pl, ow = 0, row
        gs = self.gstart.tolist()
        for g in range(len(gs) - 1):
            if gs[g] <= b < gs[g + 1]:
                pl, ow = int(self.plen[g]), int(self.owner[g])
        if n < pl:   # ends inside the prefix: reads its own pages
            pl = 0
        t = self.table.tolist()
        out = []
        for p in range(n):
            pg = t[ow if p < pl else row][p // self.page]
            if 0 <= pg < self.k.shape[0]:
                out.append((pg, p % self.page))
        return out

    def check(self, o, rows=None, scale=None):
        scale = 1 / math.sqrt(self.hd) if scale is None else scale
        u = torch.finfo(self.dtype).eps / 2
        G = self.Hq // self.Hk
        for r in (range(self.B * self.S) if rows is None else rows):
            sl = self.slots(r)
            got = o[r].double().view(self.Hk, G, self.hd)
            if not sl:
                assert not got.any(), f"row {r}: zeros expected"
                continue
            pg, of = (torch.tensor(x, device=DEV) for x in zip(*sl))
            kk, vv = self.k[pg, :, of].double().transpose(0, 1), self.v[pg, :, of].double().transpose(0, 1)
            q = self.q[r].double().view(self.Hk, G, self.hd)
            s = q @ kk.transpose(1, 2) * scale
            w = torch.softmax(s, -1)
            ref, A = w @ vv, w @ vv.abs()
            e = (q.abs() @ kk.abs().transpose(1, 2) * abs(scale)).amax(-1, keepdim=True) * self.hd * 2.0 ** -23
            n = len(sl)
            tol = u * (A + ref.abs()) + (4 * e + 2.0 ** -21 + n / 8 * 2.0 ** -23) * A
            if self.dtype == H:
                tol = tol + 2.0 ** -25 * vv.abs().sum(1, keepdim=True) + 2.0 ** -25
            d = (got - ref).abs()
            assert bool((d <= tol).all()), f"row {r} ({n} positions): worst {float((d / tol).max()):.2f} of the tolerance"


CASES = [
    # one token, one position; the smallest calls
    dict(groups=[(0, [1])], Hq=1, Hk=1),
    dict(groups=[(1, [1])], Hq=2, Hk=1, hd=64, page=16),
    dict(groups=[(1, [2, 1, 5])], Hq=2, Hk=2, hd=256, page=32),
    # ends inside, on and one past a tile and a page
    dict(groups=[(63, [63, 64, 65, 66])]),
    dict(groups=[(64, [64, 65, 127, 128, 129])], page=16, dtype=BF),
    dict(groups=[(65, [65, 66, 130])], page=32),
    dict(groups=[(100, [128, 200, 101])], page=128, hd=64),
    dict(groups=[(48, [64, 49, 112])], page=16, hd=256, dtype=BF),
    # several groups, one of them without a prefix, one with a single sequence
    dict(groups=[(130, [131, 140, 300]), (0, [7, 70]), (500, [513])], Hq=8, Hk=2),
    # rows that end inside the prefix, padding rows at the edges and a padded owner-to-be
    dict(groups=[(200, [0, 210, 3, 200, -1]), (90, [-1, 95])], Hq=3, Hk=1),
    dict(groups=[(0, [0]), (64, [0, 0])]),
    # blocks of more than 16 query rows, ragged over 64
    dict(groups=[(300, [301 + 7 * i for i in range(23)])], Hq=6, Hk=2),
    dict(groups=[(300, [301 + 7 * i for i in range(23)])], Hq=6, Hk=2, hd=256, page=16, dtype=BF),
    dict(groups=[(257, [258 + i for i in range(9)]), (64, [70, 80])], Hq=14, Hk=2, hd=64, page=32),
    # several rows a sequence, each with its own limit; more than 64 query rows a sequence
    dict(groups=[(100, [102, 130])], S=2, Hq=8, Hk=1),
    dict(groups=[(40, [45, 90, 200])], S=5, Hq=4, Hk=4, page=16),
    dict(groups=[(33, [120, 77])], S=30, Hq=8, Hk=2, page=32, dtype=BF),
    dict(groups=[(10, [40])], S=40, Hq=3, Hk=1, hd=64),
    dict(groups=[(20, [60, 3])], S=12, Hq=16, Hk=2, hd=256),          # the first rows of a sequence are padding
    # many heads a KV head
    dict(groups=[(70, [75, 71])], Hq=64, Hk=1, hd=64, page=64),
    dict(groups=[(70, [75, 71])], Hq=17, Hk=1),
    # large scores
    dict(groups=[(150, [170, 151])], amp=4.0),
    dict(groups=[(150, [170, 151])], amp=4.0, dtype=BF, hd=256),
]


@pytest.mark.parametrize("c", range(len(CASES)))
def test_matches_formula(c):
    x = Case(seed=c, **CASES[c])
    x.check(x.run())


@pytest.mark.parametrize("hd,page,dtype", [(128, 64, H), (64, 16, BF), (256, 128, H)])
def test_long_prefix(hd, page, dtype):
    """A prefix of many splits, short and long sequences behind it."""
    x = Case([(9001, [9002, 9500, 9001, 11003]), (4100, [4101, 4164])], Hq=6, Hk=2, hd=hd, page=page, dtype=dtype)
    x.check(x.run())


def test_crowd():
    x = Case([(1000, [1001 + 13 * i for i in range(64)])], Hq=8, Hk=2, page=32, dtype=BF)
    o = x.run()
    x.check(o, rows=range(0, 64, 5))
    assert torch.equal(o, x.run()), "the result does not depend on scheduling"


@pytest.mark.parametrize("hd,dtype", [(64, H), (64, BF), (128, H)])
def test_many_jobs_behind_large_blocks(hd, dtype):
    """More KV heads and groups of 65 to 128 query rows than the grid has CTAs: each takes several jobs in turn,
    and its list of them must outlive the blocks before."""
    x = Case([(1 + g, [2 + g + i for i in range(9 + g % 8)]) for g in range(36)], Hq=128, Hk=16, hd=hd, page=16,
             dtype=dtype)
    x.check(x.run(), rows=range(0, x.B, 7))


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_several_blocks_a_group_and_head(hd):
    """Groups of 128 + 40 and 128 + 48 rows a KV head on a prefix of many tiles."""
    x = Case([(1500, [1501 + 5 * i for i in range(n)]) for n in (21, 21, 22)], Hq=64, Hk=8, hd=hd, page=32)
    x.check(x.run(), rows=range(0, x.B, 3))


def test_groups_are_only_a_way_to_read():
    """With and without groups, and with the groups merged, the outputs agree to rounding."""
    x = Case([(200, [210, 333, 201]), (64, [65, 100])])
    x.check(x.run(gstart=None, owner=None, plen=None))
    empty = torch.zeros(1, dtype=torch.int32, device=DEV)
    x.check(x.run(gstart=empty, owner=empty[:0], plen=empty[:0]))
    x.gstart = torch.tensor([3, 5], dtype=torch.int32, device=DEV)     # only the second group
    x.owner, x.plen = x.owner[1:].clone(), x.plen[1:].clone()
    x.check(x.run())


def test_equals_the_flat_attention():
    """Against hm_decode_attn on the same values in a flat cache."""
    from estudiocanciones_b200 import kernels
    x = Case([(300, [310, 420, 301, 555])], Hq=24, Hk=8)
    L = 640
    kc, vc = torch.zeros(4, 8, L, 128, device=DEV).half(), torch.zeros(4, 8, L, 128, device=DEV).half()
    for b in range(4):
        for p, (pg, sl) in enumerate(x.slots(b)):
            kc[b, :, p], vc[b, :, p] = x.k[pg, :, sl], x.v[pg, :, sl]
    o = torch.empty_like(x.q)
    kernels.attn(x.q, kc, vc, x.pos, o, 1, 24, 8, L)
    torch.testing.assert_close(x.run().float(), o.float(), atol=2e-3, rtol=5e-3)


def test_strides_and_sequence_rows():
    """Row pitches of q, o and the table; sequences anywhere in the table; a given scale."""
    x = Case([(100, [110, 150]), (0, [30])], Hq=4, Hk=2)
    wide = torch.full((8, 64), -9, dtype=torch.int32, device=DEV)
    w = x.table.shape[1]
    rows = [5, 0, 7]
    for b, r in enumerate(rows):
        wide[r, 1:1 + w] = x.table[b]
    x.table = wide[:, 1:1 + w]
    x.seqs = torch.tensor(rows, dtype=torch.int32, device=DEV)
    x.owner = torch.tensor([rows[int(i)] for i in x.owner], dtype=torch.int32, device=DEV)
    buf = torch.randn(3, 4 * 128 + 64, device=DEV).half()
    x.q = buf[:, 32:-32]
    out = torch.full((3, 4 * 128 + 16), 5.0, device=DEV).half()
    o = x.run(o=out[:, 8:-8], scale=0.03)
    x.check(o, scale=0.03)
    assert bool((out[:, :8] == 5).all()) and bool((out[:, -8:] == 5).all())


def test_infinities_outside_a_rows_sight():
    """Slots past a sequence's end may hold anything, infinities too; seen ones give what the formula gives."""
    x = Case([(70, [75, 100])], Hq=2, Hk=1)
    bad = torch.isnan(x.k)
    ref = x.run()
    for val in (float("inf"), -float("inf"), 65504.0):
        x.k[bad] = val
        x.v[bad] = val
        assert torch.equal(x.run(), ref)
    pg, sl = x.slots(1)[90]
    x.v[pg, 0, sl, 3] = float("inf")
    o = x.run()
    assert torch.equal(o[0], ref[0]) and bool((o[1].view(2, 128)[:, 3] == float("inf")).all())
    x.k[pg, 0, sl] = float("nan")
    o = x.run()
    assert torch.equal(o[0], ref[0]) and bool(o[1].isnan().all())


@pytest.mark.parametrize("S,Hq,Hk,hd,page,dtype", [(2, 4, 2, 128, 64, H), (5, 3, 1, 64, 16, BF), (3, 2, 1, 256, 32, H),
                                                   (8, 4, 1, 128, 16, BF), (6, 8, 1, 128, 64, H), (40, 2, 1, 64, 32, H),
                                                   (30, 3, 1, 256, 16, BF), (100, 1, 1, 128, 32, H)])
def test_infinities_between_the_rows_of_a_sequence(S, Hq, Hk, hd, page, dtype):
    """A V (or K) that is not finite, at a position that only later rows see, reaches those alone."""
    x = Case([(70, [70 + S, 70 + S + 40, 68 + S]), (0, [S + 3])], S=S, Hq=Hq, Hk=Hk, hd=hd, page=page, dtype=dtype)
    ref = x.run()
    for b in range(4):
        n = int(x.pos[b * S + S - 1]) + 1
        for back, val in ((1, float("inf")), (S - 1, -float("inf"))):   # seen by the last row; by all but the first
            y = Case([(70, [70 + S, 70 + S + 40, 68 + S]), (0, [S + 3])], S=S, Hq=Hq, Hk=Hk, hd=hd, page=page, dtype=dtype)
            p = n - back
            if b < 3 and p < 70:   # read through the group's owner
                continue
            pg, sl = y.table[b, p // page], p % page
            y.v[pg, 0, sl, 5] = val
            o = y.run()
            for r in range(4 * S):
                sees = r // S == b and int(x.pos[r]) >= p
                row = o[r].view(Hk, Hq // Hk, hd)
                if sees:
                    assert bool((row[0, :, 5] == val).all())
                    row[0, :, 5] = 0
                else:
                    assert torch.equal(o[r], ref[r]) or bool(o[r].isfinite().all())
            y.v[pg, 0, sl, 5] = 0
            clean = y.run()
            clean.view(4 * S, Hk, Hq // Hk, hd)[b * S:(b + 1) * S, 0, :, 5] = 0
            o.view(4 * S, Hk, Hq // Hk, hd)[b * S:(b + 1) * S, 0, :, 5] = 0
            torch.testing.assert_close(o.float(), clean.float(), atol=4 * torch.finfo(dtype).eps, rtol=4 * torch.finfo(dtype).eps)
            y.k[pg, 0, sl] = float("nan")
            o = y.run()
            for r in range(4 * S):
                sees = r // S == b and int(x.pos[r]) >= p
                assert bool(o[r].view(Hk, Hq // Hk, hd)[0].isnan().all()) == sees


def test_bad_entries_are_reported_and_left_out():
    from estudiocanciones_b200 import kernels
    BAD = _lib.HM_ERR_BADINDEX

    def fresh():
        return Case([(130, [131, 190]), (64, [64, 300])], page=16)
    for entry, val in (((1, 9), 10 ** 6), ((1, 9), -1), ((1, 2), 10 ** 6), ((3, 18), -5)):   # row 1 owns the first prefix
        x = fresh()
        x.table[entry] = val                          # its positions are left out
        o = x.run()
        assert kernels.read_errors(DEV) == BAD
        x.check(o)
    for p in (10 ** 6, 2 ** 40, 19 * 16):
        x = fresh()
        x.pos[1] = p                                  # a row without a valid position: zeros
        o = x.run()
        assert kernels.read_errors(DEV) == BAD and not o[1].any()
        x.check(o, rows=[0, 2, 3])
    for name, val in (("owner", [0, 99]), ("owner", [0, -1]), ("plen", [130, -4]), ("plen", [130, 10 ** 6])):
        x = fresh()
        setattr(x, name, torch.tensor(val, dtype=torch.int32, device=DEV))
        o = x.run()
        assert kernels.read_errors(DEV) == BAD
        x.plen = torch.tensor([130, 0], dtype=torch.int32, device=DEV)   # that group reads its own pages
        x.owner = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
        x.check(o)
    for val in ([0, 3, 2], [0, 2, 5], [-1, 2, 4], [-10 ** 9, 2, 4], [10 ** 9, 2, 4], [0, -7, 10 ** 9], [4, 2, 0]):
        x = fresh()
        x.gstart = torch.tensor(val, dtype=torch.int32, device=DEV)
        o = x.run()
        assert kernels.read_errors(DEV) == BAD
        x.gstart, x.plen = torch.tensor([0, 0, 0], dtype=torch.int32, device=DEV), torch.zeros_like(x.plen)
        x.check(o)                                    # no groups at all
    x = fresh()
    x.seqs = torch.tensor([0, 4, 2, 3], dtype=torch.int32, device=DEV)
    o = x.run()
    assert kernels.read_errors(DEV) == BAD and not o[1].any()
    x.check(o, rows=[0, 2, 3])


def test_captured_call_follows_the_lengths():
    """One graph; positions, prefix lengths and pages change between replays."""
    from estudiocanciones_b200._lib import capture_graph
    x = Case([(128, [300, 290, 310]), (64, [100])], page=32)
    x.run()
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with capture_graph(g, s):
        o = x.run()
    for pos, plen in (([299, 289, 309, 99], [128, 64]), ([150, 128, 127, 63], [96, 0]), ([-1, 5, 200, 70], [128, 64]),
                      ([-1, -1, -1, -1], [0, 0])):
        x.pos.copy_(torch.tensor(pos, device=DEV))
        x.plen.copy_(torch.tensor(plen, dtype=torch.int32, device=DEV))
        g.replay()
        x.check(o)
    del g


def test_two_calls_at_once():
    """Calls on two streams do not share scratch."""
    a, b = Case([(900, [1000, 901])], seed=1), Case([(640, [700, 1000, 641])], seed=2, page=16)
    ra, rb = a.run(), b.run()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(10):
        with torch.cuda.stream(sa):
            outs.append((a.run(), ra))
        with torch.cuda.stream(sb):
            outs.append((b.run(), rb))
    torch.cuda.synchronize()
    assert all(torch.equal(o, r) for o, r in outs)


def test_pool_rows_past_32_bit_bytes():
    """Pages whose byte offset passes 2^32."""
    k = torch.zeros(70000, 4, 64, 128, device=DEV, dtype=H)           # 4.6 GB
    v = torch.zeros_like(k)
    x = Case([(100, [120, 180])], Hq=8, Hk=4)
    top = k.shape[0] - x.k.shape[0]
    k[top:], v[top:] = x.k, x.v
    x.table = torch.where(x.table >= 0, x.table + top, x.table)
    x.k, x.v = k, v
    x.check(x.run())


def test_refused_arguments():
    x = Case([(100, [110, 150])], Hq=4, Hk=2)
    f16 = x.q
    for kw in (dict(S=3), dict(S=0), dict(plen=None), dict(gstart=None), dict(plen=x.plen.long()), dict(owner=x.owner[:0]),
               dict(o=torch.empty(2, 4 * 128, device=DEV)), dict(o=torch.empty(2, 4 * 128 + 8, device=DEV, dtype=H)),
               dict(seqs=torch.zeros(3, dtype=torch.int32, device=DEV)), dict(plen=x.plen.cpu())):
        with pytest.raises(HMError):
            x.run(**kw)
    for name, val in (("q", f16[:, :-8]), ("q", f16.bfloat16()), ("q", f16.cpu()), ("q", f16.t()), ("q", f16[:, :128]),
                      ("k", x.k[:, :, :, :64]), ("k", x.k.bfloat16()), ("table", x.table.long()), ("table", x.table[:1]),
                      ("table", x.table.t()), ("pos", x.pos.int()), ("pos", x.pos[:1])):
        y = Case([(100, [110, 150])], Hq=4, Hk=2)
        setattr(y, name, val)
        with pytest.raises(HMError):
            y.run()
    for hd, page in ((96, 64), (128, 24), (128, 8), (128, 96)):
        k = torch.zeros(4, 2, page, hd, device=DEV, dtype=H)
        y = Case([(10, [11])], Hq=4, Hk=2)
        y.k, y.v, y.q = k, k.clone(), torch.zeros(1, 4 * hd, device=DEV, dtype=H)
        with pytest.raises(HMError):
            y.run()
    y = Case([(10, [11])], Hq=4, Hk=2)
    y.q = torch.zeros(1, 4 * 128 + 8, device=DEV, dtype=H)[:, 4:-4]    # rows that do not start on 16 bytes
    with pytest.raises(HMError):
        y.run()
