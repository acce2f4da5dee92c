"""Cache pages: grow, fork, free, copy, compact and the paged RoPE/KV write against a host
model of the same rules (whole numbers and moved data equal, rotated values within the types'
rounding)."""
import random

import pytest
import torch

from estudiocanciones_b200 import _lib
from estudiocanciones_b200._lib import HMError

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _built():
    from estudiocanciones_b200 import build, kernels
    build.build()
    kernels.read_errors(DEV)
    yield
    assert kernels.read_errors(DEV) == 0, "a kernel reported an error bit"


class Model:
    """The rules on host lists."""

    def __init__(self, pool):
        self.page = pool.page
        self.k, self.v = pool.k.cpu().clone(), pool.v.cpu().clone()
        self.table = pool.table.tolist()
        self.lens = pool.lens.tolist()
        self.refs = pool.refs.tolist()

    def held(self, n):
        return -(-n // self.page)

    def grow(self, seqs, n):
        need = sum(self.held(self.lens[s] + n) - self.held(self.lens[s]) for s in seqs)
        if need > self.refs.count(0):
            return False
        for s in seqs:
            for j in range(self.held(self.lens[s]), self.held(self.lens[s] + n)):
                p = self.refs.index(0)
                self.refs[p], self.table[s][j] = 1, p
            self.lens[s] += n
        return True

    def fork(self, src, dst):
        if sum(self.lens[a] % self.page > 0 for a in src) > self.refs.count(0):
            return False
        for a, b in zip(src, dst):
            self.lens[b] = self.lens[a]
            for j in range(self.lens[a] // self.page):
                self.table[b][j] = self.table[a][j]
                self.refs[self.table[a][j]] += 1
        for a, b in zip(src, dst):
            j, part = divmod(self.lens[a], self.page)
            if part:
                p, q = self.refs.index(0), self.table[a][j]
                self.refs[p], self.table[b][j] = 1, p
                for t in (self.k, self.v):
                    t[:, p, :, :part] = t[:, q, :, :part]
        return True

    def free(self, seqs):
        for s in seqs:
            for p in self.table[s]:
                if p >= 0:
                    self.refs[p] -= 1
            self.table[s] = [-1] * len(self.table[s])
            self.lens[s] = 0

    def copy(self, src, dst):
        for t in (self.k, self.v):
            t[:, dst] = t[:, src]

    def compact(self):
        n = sum(r > 0 for r in self.refs)
        to = dict(zip([p for p in range(n, len(self.refs)) if self.refs[p] > 0],
                      [p for p in range(n) if self.refs[p] == 0]))
        for a, b in to.items():
            for t in (self.k, self.v):
                t[:, b] = t[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        return n

    def check(self, pool):
        assert pool.table.tolist() == self.table
        assert pool.lens.tolist() == self.lens
        assert pool.refs.tolist() == self.refs
        assert torch.equal(pool.k.cpu(), self.k) and torch.equal(pool.v.cpu(), self.v)


def make(layers=2, n_pages=40, Hk=2, hd=64, max_seqs=12, max_len=200, page=16, dtype=torch.float16, seed=0):
    from estudiocanciones_b200.pages import PagePool
    pool = PagePool(layers, n_pages, Hk, hd, max_seqs, max_len, page, dtype, DEV)
    g = torch.Generator().manual_seed(seed)
    for t in (pool.k, pool.v):
        t.copy_(torch.randn(t.shape, generator=g).to(dtype))
    return pool, Model(pool)


@pytest.mark.parametrize("seed,page,hd,dtype", [(0, 16, 64, torch.float16), (1, 32, 128, torch.bfloat16),
                                                (2, 64, 256, torch.float16), (3, 1, 8, torch.float16),
                                                (4, 128, 128, torch.float16), (5, 7, 24, torch.bfloat16)])
def test_random_life_of_a_pool(seed, page, hd, dtype):
    """A long random run of calls keeps table, lens, refs and every byte of the pool equal to the model's."""
    rng = random.Random(seed)
    pool, m = make(page=page, hd=hd, dtype=dtype, seed=seed, max_len=12 * page, n_pages=50, layers=rng.randint(1, 3),
                   Hk=rng.randint(1, 3))
    from estudiocanciones_b200 import kernels
    for step in range(60):
        live = [s for s in range(12) if m.lens[s] > 0]
        empty = [s for s in range(12) if m.lens[s] == 0]
        op = rng.choice(["grow", "grow", "fork", "free", "compact", "copy"])
        ok = True
        if op == "grow":
            n = rng.choice([0, 1, 1, page, rng.randint(1, 3 * page)])
            seqs = [s for s in rng.sample(range(12), rng.randint(1, 5)) if m.lens[s] + n <= 12 * page]
            if seqs:
                pool.grow(seqs, n)
                ok = m.grow(seqs, n)
        elif op == "fork" and live and empty:
            dst = rng.sample(empty, rng.randint(1, min(4, len(empty))))
            src = [rng.choice(live) for _ in dst]
            pool.fork(src, dst)
            ok = m.fork(src, dst)
        elif op == "free" and len(live) > 3:
            seqs = rng.sample(live, 2)
            pool.free(seqs)
            m.free(seqs)
        elif op == "compact":
            assert int(pool.compact()) == m.compact()
        elif op == "copy":
            ids = rng.sample(range(50), 6)
            pool.copy(ids[:3], ids[3:])
            m.copy(ids[:3], ids[3:])
        assert kernels.read_errors(DEV) == (0 if ok else _lib.HM_ERR_NOPAGES)
        m.check(pool)


def test_refused_lists_change_nothing():
    from estudiocanciones_b200 import kernels
    pool, m = make(max_len=64)
    pool.grow([0, 1], 20)
    m.grow([0, 1], 20)
    bad = [lambda: pool.grow([2, 2], 1), lambda: pool.grow([12], 1), lambda: pool.grow([0], 45),
           lambda: pool.free([1, 1]), lambda: pool.free([0, 99]), lambda: pool.fork([0], [1]),
           lambda: pool.fork([0, 1], [2, 2]), lambda: pool.fork([2, 0], [3, 2]), lambda: pool.fork([0], [12]),
           lambda: pool.fork([-1], [3]), lambda: pool.fork([3], [3]), lambda: pool.copy([0, 1], [2, 2]),
           lambda: pool.copy([0, 2], [2, 3]), lambda: pool.copy([0], [40]), lambda: pool.copy([-1], [4])]
    for f in bad:
        f()
        assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX
        m.check(pool)
    pool.grow([3, 4, 5, 6, 7, 8, 9, 10, 11], 64)   # 36 pages, 36 free: fits exactly
    assert kernels.read_errors(DEV) == 0 and pool.free_pages() == 0
    before = pool.table.clone()
    pool.grow([2], 1)
    assert kernels.read_errors(DEV) == _lib.HM_ERR_NOPAGES and torch.equal(pool.table, before)
    pool.fork([0], [2])                              # its partial page needs a free one
    assert kernels.read_errors(DEV) == _lib.HM_ERR_NOPAGES and torch.equal(pool.table, before)


def test_disagreeing_tables_are_reported():
    from estudiocanciones_b200 import kernels
    pool, m = make()
    pool.grow([0], 20)
    pool.table[0, 1] = 1000                          # no such page
    pool.fork([0], [1])
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and int(pool.lens[1]) == 0
    pool.grow([0], 1)
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and int(pool.lens[0]) == 20
    pool.free([0])
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and int(pool.lens[0]) == 20
    pool.compact()
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX
    pool.table[0, 1] = 1
    pool.refs[1] = 2                                 # a partial page that two sequences hold
    pool.grow([0], 1)
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and int(pool.lens[0]) == 20


def snapshot(pool):
    return [t.clone() for t in (pool.k, pool.v, pool.table, pool.lens, pool.refs)]


def unchanged(pool, before):
    return all(torch.equal(a, b) for a, b in zip(snapshot(pool), before))


def test_rows_that_hold_more_than_the_counts_say_are_not_freed():
    """A page counted once that two listed rows, or one row twice, name: the call changes nothing."""
    from estudiocanciones_b200 import kernels
    pool, m = make()
    pool.grow([0, 1, 2], 40)
    m.grow([0, 1, 2], 40)
    right = pool.table.clone()
    pool.table[1, 2] = pool.table[0, 1]
    before = snapshot(pool)
    for seqs in ([0, 1], [1, 0], [2, 1, -1, 0]):
        pool.free(seqs)
        assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and unchanged(pool, before)
    pool.table.copy_(right)
    pool.table[2, 0] = pool.table[2, 1]
    before = snapshot(pool)
    pool.free([0, 2])
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and unchanged(pool, before)
    pool.table.copy_(right)
    pool.fork([0], [3])                              # two full pages that two rows hold, and are counted twice
    m.fork([0], [3])
    pool.free([0, 3, 1])
    m.free([0, 3, 1])
    assert kernels.read_errors(DEV) == 0
    m.check(pool)


@pytest.mark.parametrize("stale", [2, 7, 20, 40, 1000])
def test_compaction_checks_the_table_first(stale):
    """An entry that names a page nobody holds (below the live count, above it) or none of the pool's: nothing
    changes, and the count returned is the pool's size, below which every live page lies."""
    from estudiocanciones_b200 import kernels
    pool, m = make()
    pool.grow([0, 1, 2, 3], 32)
    pool.free([1, 3])                                # live 0 1 4 5 -> 0 1 2 3; 2 3 6 7 and up are free
    m.grow([0, 1, 2, 3], 32)
    m.free([1, 3])
    pool.table[9, 5] = stale
    before = snapshot(pool)
    n = pool.compact()
    assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and unchanged(pool, before) and int(n) == 40
    pool.table[9, 5] = -1
    assert int(pool.compact()) == m.compact() == 4
    assert kernels.read_errors(DEV) == 0
    m.check(pool)


def test_skipped_entries():
    pool, m = make()
    pool.grow([-1, 0, -5, 3], 17)
    m.grow([0, 3], 17)
    pool.fork([0, 7, 3], [1, -1, 2])
    m.fork([0, 3], [1, 2])
    pool.free([-1, 0])
    m.free([0])
    m.check(pool)
    pool.copy([0, 99, 3], [30, -1, 31])
    m.copy([0, 3], [30, 31])
    m.check(pool)


def test_long_lists_and_a_wide_pool():
    """1024 sequences at once; more pages than one round of the bookkeeping reads."""
    from estudiocanciones_b200.pages import PagePool
    n = 20000
    pool = PagePool(1, n, 1, 8, 1100, 40, 2, torch.float16, DEV)
    g = torch.Generator().manual_seed(1)
    taken = torch.rand(n, generator=g) < 0.4
    pool.refs.copy_(taken.int())
    seqs = torch.randperm(1100, generator=g)[:1024].int()
    pool.grow(seqs.to(DEV), 13)                      # 7 pages each
    free = (~taken).nonzero().flatten()
    want = free[:7 * 1024].view(1024, 7)
    assert torch.equal(pool.table.cpu()[seqs.long(), :7], want.int())
    assert int((pool.refs > 0).sum()) == int(taken.sum()) + 7 * 1024
    refs = pool.refs.cpu()
    old = pool.k.clone()
    n_live = int(pool.compact())
    assert n_live == int((refs > 0).sum()) and bool((pool.refs[:n_live] == 1).all()) and not pool.refs[n_live:].any()
    del old
    at = torch.arange(n)
    to = at.clone()
    to[(refs > 0) & (at >= n_live)] = at[(refs == 0) & (at < n_live)]
    assert torch.equal(pool.table.cpu()[seqs.long(), :7], to[want].int())


def test_compaction_of_a_wide_pool_moves_the_bytes():
    """Several rounds of counts; every moved page's K and V stand behind its new number, the others stay."""
    from estudiocanciones_b200.pages import PagePool
    n = 40000
    pool = PagePool(2, n, 2, 8, 900, 40, 2, torch.float16, DEV)
    g = torch.Generator().manual_seed(4)
    for t in (pool.k, pool.v):
        t.copy_(torch.randn(t.shape, generator=g))
    live = torch.randperm(n, generator=g)[:900 * 20].view(900, 20)
    pool.table.copy_(live)
    pool.refs[live.flatten().to(DEV)] = 1
    old_k, old_v, at = pool.k[:, live.flatten()], pool.v[:, live.flatten()], live.flatten()
    assert int(pool.compact()) == 18000
    new = pool.table.flatten().long()
    assert torch.equal(new.sort().values.cpu(), torch.arange(18000)) and int((new.cpu() != at).sum()) == int((at >= 18000).sum())
    assert torch.equal(pool.k[:, new], old_k) and torch.equal(pool.v[:, new], old_v)


@pytest.mark.parametrize("n_seqs,max_pages,n_pages", [(1, 1, 4), (1, 5000, 64), (70, 33, 300), (5, 1500, 20000), (1100, 20, 64),
                                                      (3, 1025, 64), (33, 32, 16385)])
def test_compaction_looks_at_every_cell(n_seqs, max_pages, n_pages):
    """One stale entry anywhere in tables of all shapes, in pools of one and of several rounds, is found."""
    from estudiocanciones_b200 import kernels
    from estudiocanciones_b200.pages import PagePool
    rng = random.Random(n_seqs + max_pages)
    pool = PagePool(1, n_pages, 1, 8, n_seqs, max_pages, 1, torch.float16, DEV)
    pool.refs[n_pages // 2:] = 1
    pool.table.copy_(torch.randint(n_pages // 2, n_pages, pool.table.shape, dtype=torch.int32))
    before = snapshot(pool)
    ends = [(0, 0), (n_seqs - 1, max_pages - 1), (0, max_pages - 1), (n_seqs - 1, 0)]
    for at in ends + [(rng.randrange(n_seqs), rng.randrange(max_pages)) for _ in range(20)]:
        right = int(pool.table[at])
        pool.table[at] = rng.choice([rng.randrange(n_pages // 2), n_pages, n_pages + 7])
        n = pool.compact()
        assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX and int(n) == n_pages
        pool.table[at] = right
        assert unchanged(pool, before)
    n = n_pages - n_pages // 2
    assert int(pool.compact()) == n and kernels.read_errors(DEV) == 0
    old, hole = before[2].long(), torch.arange(n_pages // 2, device=DEV)   # page i of the upper half above n goes to hole i
    moved = torch.where(old >= n, hole[(old - n).clamp(0, len(hole) - 1)], old)
    assert torch.equal(pool.table.long(), moved)


def test_captured_calls_replay():
    """grow + fork + free in one graph: every replay does the work on the state it finds."""
    from estudiocanciones_b200._lib import capture_graph
    pool, m = make(n_pages=60)
    src, dst = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in ([0, 0], [3, 4]))
    one = torch.tensor([0], dtype=torch.int32, device=DEV)
    pool.grow(one, 5)
    m.grow([0], 5)
    g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    with capture_graph(g, s):
        pool.grow(one, 9)
        pool.fork(src, dst)
        n_live = pool.compact()
        pool.free(dst)
    for _ in range(4):
        g.replay()
        m.grow([0], 9)
        m.fork([0, 0], [3, 4])
        assert int(n_live) == m.compact()
        m.free([3, 4])
        m.check(pool)
    del g


def test_another_stream_and_padded_tables():
    """Calls go to the current stream; the table may be a wider buffer's columns."""
    from estudiocanciones_b200 import kernels
    pool, m = make()
    wide = torch.full((12, 40), -7, dtype=torch.int32, device=DEV)
    wide[:, 3:16] = -1
    table = wide[:, 3:16]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        kernels.pages_grow(table, pool.lens, pool.refs, pool.page, [4, 0], 33)
        kernels.pages_fork(pool.k, pool.v, table, pool.lens, pool.refs, [4], [1])
        kernels.pages_free(table, pool.lens, pool.refs, [0])
        kernels.pages_compact(pool.k, pool.v, table, pool.refs)
    s.synchronize()
    m.grow([4, 0], 33)
    m.fork([4], [1])
    m.free([0])
    m.compact()
    pool.table.copy_(table)
    m.check(pool)
    assert bool((wide[:, :3] == -7).all()) and bool((wide[:, 16:] == -7).all())


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes: pages at its end are copied where they belong."""
    from estudiocanciones_b200.pages import PagePool
    pool = PagePool(3, 12000, 4, 128, 4, 256, 64, torch.float16, DEV)   # 2.4 GB each of K and V
    last = torch.randn(3, 4, 64, 128, device=DEV).half()
    pool.k[:, 11999] = last
    pool.v[:, 11999] = -last
    pool.copy([11999], [11000])
    assert torch.equal(pool.k[:, 11000], last) and torch.equal(pool.v[:, 11000], -last)
    pool.refs[11999] = 1
    pool.table[2, 0] = 11999
    assert int(pool.compact()) == 1 and int(pool.table[2, 0]) == 0
    assert torch.equal(pool.k[:, 0], last) and torch.equal(pool.v[:, 0], -last)


# ----------------------------------------------------------------------------- RoPE and write
@pytest.mark.parametrize("S,Hq,Hk,hd,page,dtype", [
    (1, 3, 1, 128, 16, torch.float16), (5, 4, 2, 64, 32, torch.bfloat16), (33, 6, 2, 128, 64, torch.float16),
    (70, 2, 2, 256, 16, torch.bfloat16), (2, 8, 4, 8, 1, torch.float16)])
def test_rope_pages_matches_formula(S, Hq, Hk, hd, page, dtype):
    """q and k within half a step of the type of the 64-bit rotation (plus the 32-bit products'
    own rounding: three operations of half a step 2^-24 on terms of at most |x0| + |x1|); v copied;
    every other slot of the pool untouched."""
    from estudiocanciones_b200 import kernels
    from estudiocanciones_b200.rope import rope_table
    gen = torch.Generator().manual_seed(S + hd)
    B, L = 3, 200
    pool, _ = make(Hk=Hk, hd=hd, page=page, dtype=dtype, n_pages=-(-L // page) * B + 3, max_len=L, layers=1)
    pool.grow([2, 0, 1], 150)
    seqs = torch.tensor([1, 2, 0], dtype=torch.int32, device=DEV)
    k, v = pool.layer(0)
    k0, v0 = k.clone(), v.clone()
    buf = torch.randn(B * S, (Hq + 2 * Hk) * hd + 16, generator=gen).to(dtype).to(DEV)
    qkv = buf[:, 8:-8]                                # row pitch wider than the row
    start = [0, 40, 150 - S]
    pos = torch.tensor([n + s for n in start for s in range(S)], device=DEV)
    pos[0] = -1                                       # a padding row
    q = torch.full((B * S, Hq * hd), 7.0, dtype=dtype, device=DEV)
    rope = rope_table(hd, L).to(DEV)
    kernels.rope_pages(qkv, rope, pos, q, k, v, pool.table, S, Hq, Hk, seqs)
    assert kernels.read_errors(DEV) == 0
    x = qkv.double().cpu().view(B * S, Hq + 2 * Hk, hd)
    t = torch.view_as_complex(rope.double().cpu())[pos.cpu().clamp(min=0)]
    pair = x[:, :Hq + Hk].reshape(B * S, Hq + Hk, hd // 2, 2).contiguous()
    y = torch.view_as_real(torch.view_as_complex(pair) * t[:, None]).reshape(B * S, Hq + Hk, hd)
    mag = pair.abs().sum(-1, keepdim=True).expand_as(pair).reshape(y.shape)
    tol = torch.finfo(dtype).eps / 2 * y.abs() + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps + \
        3 * 2.0 ** -24 * (1 + torch.finfo(dtype).eps) * mag
    got = q.double().cpu().view(B * S, Hq, hd)
    assert not got[0].any()
    assert bool(((got[1:] - y[1:, :Hq]).abs() <= tol[1:, :Hq]).all())
    table, kk, vv = pool.table.tolist(), k.cpu(), v.cpu()
    touched = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for r in range(1, B * S):
        p = int(pos[r])
        pg, sl = table[int(seqs[r // S])][p // page], p % page
        touched[pg, sl] = True
        assert bool(((kk[pg, :, sl].double() - y[r, Hq:]).abs() <= tol[r, Hq:]).all())
        assert torch.equal(vv[pg, :, sl].double(), x[r, Hq + Hk:])
    keep = ~touched[:, None, :, None].expand_as(kk)
    assert torch.equal(kk[keep], k0.cpu()[keep]) and torch.equal(vv[keep], v0.cpu()[keep])


def test_rope_pages_equals_the_flat_cache():
    """Bit for bit the values that rope_cache writes into a flat cache."""
    from estudiocanciones_b200 import kernels
    from estudiocanciones_b200.rope import rope_table
    gen = torch.Generator().manual_seed(9)
    B, S, Hq, Hk, hd, L = 2, 37, 6, 2, 128, 64
    pool, _ = make(Hk=Hk, hd=hd, page=16, n_pages=20, max_len=L, layers=1)
    pool.grow([0, 1], L)
    qkv = torch.randn(B * S, (Hq + 2 * Hk) * hd, generator=gen).half().to(DEV)
    pos = (torch.arange(S).repeat(B) + 11).to(DEV)
    rope = rope_table(hd, L).to(DEV)
    kc, vc = torch.zeros(B, Hk, L, hd, device=DEV).half(), torch.zeros(B, Hk, L, hd, device=DEV).half()
    q1, q2 = torch.empty(B * S, Hq * hd, device=DEV).half(), torch.empty(B * S, Hq * hd, device=DEV).half()
    kernels.rope_cache(qkv, rope, pos, q1, kc, vc, S, Hq, Hk, L)
    k, v = pool.layer(0)
    kernels.rope_pages(qkv, rope, pos, q2, k, v, pool.table, S, Hq, Hk)
    assert torch.equal(q1, q2)
    flat = k[pool.table[:B].long()].permute(0, 2, 1, 3, 4).reshape(B, Hk, L, hd)
    flat_v = v[pool.table[:B].long()].permute(0, 2, 1, 3, 4).reshape(B, Hk, L, hd)
    assert torch.equal(flat[:, :, 11:11 + S], kc[:, :, 11:11 + S])
    assert torch.equal(flat_v[:, :, 11:11 + S], vc[:, :, 11:11 + S])


def test_rope_pages_reports_missing_pages():
    from estudiocanciones_b200 import kernels
    pool, _ = make(layers=1)
    pool.grow([0], 16)
    k, v = pool.layer(0)
    k0 = k.clone()
    rope = torch.zeros(300, 32, 2, device=DEV)
    qkv = torch.ones(1, 6 * 64, device=DEV).half()
    q = torch.empty(1, 2 * 64, device=DEV).half()
    for p, seq in ((16, 0), (0, 1), (250, 0), (10 ** 12, 0), (0, 77), (0, -1)):
        pos, seqs = torch.tensor([p], device=DEV), torch.tensor([seq], dtype=torch.int32, device=DEV)
        kernels.rope_pages(qkv, rope, pos, q, k, v, pool.table, 1, 2, 2, seqs)
        assert kernels.read_errors(DEV) == _lib.HM_ERR_BADINDEX
        assert torch.equal(k, k0) and not q.any()


def test_refused_arguments():
    from estudiocanciones_b200 import kernels
    pool, _ = make(layers=1)
    k, v = pool.layer(0)
    for f in (lambda: pool.grow([], 1), lambda: pool.grow([0], -1), lambda: pool.grow(list(range(1025)), 1),
              lambda: pool.grow(torch.tensor([0], device=DEV), 1), lambda: pool.fork([0], [1, 2]),
              lambda: pool.fork([0], torch.tensor([1], dtype=torch.int32)),
              lambda: kernels.pages_grow(pool.table.long(), pool.lens, pool.refs, 16, [0]),
              lambda: kernels.pages_grow(pool.table.t(), pool.lens, pool.refs, 16, [0]),
              lambda: kernels.pages_grow(pool.table, pool.lens.int(), pool.refs, 16, [0]),
              lambda: kernels.pages_grow(pool.table, pool.lens, pool.refs, 0, [0]),
              lambda: kernels.pages_free(pool.table, pool.lens, pool.refs.cpu(), [0]),
              lambda: kernels.pages_compact(pool.k, pool.v, pool.table, pool.refs[:-1]),
              lambda: kernels.pages_copy(pool.k[:, ::2], pool.v[:, ::2], [0], [1]),
              lambda: kernels.pages_copy(pool.k, pool.v.bfloat16(), [0], [1])):
        with pytest.raises(HMError):
            f()
