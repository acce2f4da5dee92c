"""The serving operators together, as a program uses them: a prompt through the 8-bit product into
pages, forked to takes that read it once for all, against the same network on the flat cache; the
prompt pass with 8-bit activations; the torch.library operators."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(scope="module", autouse=True)
def _built():
    from estudiocanciones_b200 import build, kernels
    build.build()
    kernels.read_errors(DEV)
    yield
    assert kernels.read_errors(DEV) == 0, "a kernel reported an error bit"


class Net:
    """A small stack of decoder layers with int8 weights."""

    def __init__(self, layers=2, D=256, Hq=4, Hk=2, hd=128, F=512, seed=0):
        g = torch.Generator().manual_seed(seed)

        def lin(n, k):
            w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
            return w.to(DEV), torch.full((n,), 1 / (73 * k ** 0.5)).half().to(DEV)
        self.D, self.Hq, self.Hk, self.hd = D, Hq, Hk, hd
        self.layers = [dict(qkv=lin((Hq + 2 * Hk) * hd, D), o=lin(D, Hq * hd), w13=lin(2 * F, D), w2=lin(D, F),
                            n1=(1 + 0.1 * torch.randn(D, generator=g)).half().to(DEV),
                            n2=(1 + 0.1 * torch.randn(D, generator=g)).half().to(DEV)) for _ in range(layers)]
        from estudiocanciones_b200.rope import rope_table
        self.rope = rope_table(hd, 512).to(DEV)

    def run(self, x, attention):
        """x [R, D]; attention(layer, qkv) -> [R, Hq * hd] writes the cache and attends."""
        from estudiocanciones_b200 import kernels as K
        for i, L in enumerate(self.layers):
            o = attention(i, K.int8_mm_a8(K.rms(x, L["n1"]), *L["qkv"]))
            x = K.int8_mm_a8(o, *L["o"], res=x)
            m = K.int8_mm_a8(K.rms(x, L["n2"]), *L["w13"], silu=True)
            x = K.int8_mm_a8(m, *L["w2"], res=x)
        return x


def paged(net, pool, pos, S, seqs, groups):
    from estudiocanciones_b200 import kernels as K

    def attention(i, qkv):
        k, v = pool.layer(i)
        q = torch.empty(qkv.shape[0], net.Hq * net.hd, device=DEV, dtype=qkv.dtype)
        K.rope_pages(qkv, net.rope, pos, q, k, v, pool.table, S, net.Hq, net.Hk, seqs)
        return K.prefix_attn(q, k, v, pool.table, pos, *groups, S=S, seqs=seqs)
    return attention


def flat(net, kc, vc, pos, S, L):
    from estudiocanciones_b200 import kernels as K

    def attention(i, qkv):
        R = qkv.shape[0]
        q = torch.empty(R, net.Hq * net.hd, device=DEV, dtype=qkv.dtype)
        K.rope_cache(qkv, net.rope, pos, q, kc[i], vc[i], S, net.Hq, net.Hk, L)
        if S > 1:
            return K.prefill_attn(q, kc[i], vc[i], S)
        o = torch.empty_like(q)
        K.attn(q, kc[i], vc[i], pos, o, 1, net.Hq, net.Hk, L)
        return o
    return attention


@pytest.mark.parametrize("P,page", [(70, 16), (128, 64), (200, 32)])
def test_takes_of_two_prompts(P, page):
    """Two prompts, three takes each, eight frames in one captured graph: hidden states follow the flat
    cache's (whose rows each hold and read their own copy of the prompt).

    The two paths differ in the attention's summation order alone: about two fp16 steps of an output,
    which the next layer's token quantisation can turn into whole steps of 1/127 of a row's largest
    value on single elements; over two layers and 256-wide sums that stays within a few per cent of
    the norm."""
    from estudiocanciones_b200._lib import capture_graph
    from estudiocanciones_b200.pages import PagePool
    net = Net()
    g = torch.Generator().manual_seed(P)
    n, frames, L = 3, 8, 512
    prompts = torch.randn(2 * P, net.D, generator=g).half().to(DEV)
    steps = torch.randn(frames, 2 * n, net.D, generator=g).half().to(DEV)
    # flat: 6 rows, each with its prompt
    kc = [torch.zeros(2 * n, net.Hk, L, net.hd, device=DEV).half() for _ in net.layers]
    vc = [torch.zeros_like(k) for k in kc]
    rows = prompts.view(2, 1, P, net.D).expand(2, n, P, net.D).reshape(2 * n * P, net.D).contiguous()
    ppos = torch.arange(P, device=DEV).repeat(2 * n)
    ref = [net.run(rows, flat(net, kc, vc, ppos, P, L)).view(2 * n, P, net.D)[:, -1]]
    for f in range(frames):
        pos = torch.full((2 * n,), P + f, device=DEV)
        ref.append(net.run(steps[f], flat(net, kc, vc, pos, 1, L)))
    # pages: sequences 0, 1 hold the prompts, 2 .. 7 the takes
    pool = PagePool(len(net.layers), 64, net.Hk, net.hd, 10, L, page, torch.float16, DEV)
    pool.grow([0, 1], P)
    two = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    x = net.run(prompts, paged(net, pool, torch.arange(P, device=DEV).repeat(2), P, two, ()))
    takes = torch.arange(2, 2 + 2 * n, dtype=torch.int32, device=DEV)
    pool.fork(two.repeat_interleave(n), takes)
    assert int((pool.refs > 1).sum()) == 2 * (P // page)
    groups = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, n, 2 * n], [0, 1], [P, P])]
    out = [x.view(2, P, net.D)[:, -1].repeat_interleave(n, 0)]
    pos = torch.full((2 * n,), P - 1, device=DEV)
    xin = torch.zeros(2 * n, net.D, device=DEV).half()

    def frame():
        pos.add_(1)
        pool.grow(takes, 1)
        return net.run(xin, paged(net, pool, pos, 1, takes, groups))
    gr, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with capture_graph(gr, st):
        y = frame()
    for f in range(frames):
        if f == 4:   # the pool is packed in the middle of the song; the owners keep their rows
            pool.copy([60], [61])
            pool.compact()
        xin.copy_(steps[f])
        gr.replay()
        out.append(y.clone())
    del gr
    for a, b in zip(out, ref):
        err = float((a.float() - b.float()).norm() / b.float().norm())
        assert err < 0.05, err
    assert pool.lens.tolist() == [P, P] + [P + frames] * (2 * n) + [0, 0]
    # the cache itself: every take's keys and values next to the flat cache's
    for i in range(len(net.layers)):
        for b in range(2 * n):
            t = pool.table[2 + b][:-(-(P + frames) // page)].long()
            k = pool.k[i][t].transpose(0, 1).reshape(net.Hk, -1, net.hd)[:, :P + frames].float()
            d = (k - kc[i][b, :, :P + frames].float()).norm() / k.norm()
            assert float(d) < 0.05
    pool.free(takes)
    pool.free([0, 1])
    assert pool.free_pages() == 64 and bool((pool.table == -1).all())


def test_takes_go_on_after_their_pages_move():
    """A sequence in front of the takes ends in the middle of the song and its room is closed: the captured frame
    gives bit for bit what it gives in a pool where nothing moves."""
    from estudiocanciones_b200._lib import capture_graph
    from estudiocanciones_b200.pages import PagePool
    net = Net()
    P, page, frames, L = 70, 16, 14, 512
    g = torch.Generator().manual_seed(11)
    prompts = torch.randn(2 * P, net.D, generator=g).half().to(DEV)
    steps = torch.randn(frames, 4, net.D, generator=g).half().to(DEV)
    two = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    takes = torch.tensor([2, 3, 4, 5], dtype=torch.int32, device=DEV)
    groups = [torch.tensor(t, dtype=torch.int32, device=DEV) for t in ([0, 2, 4], [0, 1], [P, P])]

    def song(moves):
        pool = PagePool(len(net.layers), 64, net.Hk, net.hd, 10, L, page, torch.float16, DEV)
        pool.grow([8], 100)                                  # in front of everything
        pool.grow([0, 1], P)
        net.run(prompts, paged(net, pool, torch.arange(P, device=DEV).repeat(2), P, two, ()))
        pool.fork(two.repeat_interleave(2), takes)
        pos = torch.full((4,), P - 1, device=DEV)
        xin = torch.zeros(4, net.D, device=DEV).half()

        def frame():
            pos.add_(1)
            pool.grow(takes, 1)
            return net.run(xin, paged(net, pool, pos, 1, takes, groups))
        gr, st = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        with capture_graph(gr, st):
            y = frame()
        out = []
        for f in range(frames):
            if f == 4 and moves:
                before, used = pool.table.clone(), pool.k.shape[1] - pool.free_pages()
                pool.free([8])
                assert int(pool.compact()) == used - 7
                assert int((pool.table[:6] != before[:6]).sum()) > 0
            xin.copy_(steps[f])
            gr.replay()
            out.append(y.clone())
        del gr
        return torch.stack(out)
    assert torch.equal(song(True), song(False))


def test_prompt_pass_with_8_bit_activations():
    """prefill_backbone(a8=True) is the layer loop written out with int8_mm_a8, and makes no fp16 copies."""
    from estudiocanciones_b200 import kernels as K
    from estudiocanciones_b200.checkpoint import TINY_SHAPE, synthetic_tensors
    from estudiocanciones_b200.engine import HeartMuLaLite
    from estudiocanciones_b200.prefill import prefill_backbone
    t = synthetic_tensors(TINY_SHAPE, seed=5, gamma_one=False)
    m = HeartMuLaLite(t, device=DEV, bb_heads=TINY_SHAPE.bb_heads, dec_heads=TINY_SHAPE.dec_heads)
    B, P, L = 2, 45, 64
    m.alloc(1, B, L)
    h = m.text_emb(torch.randint(0, 1024, (B, P), device=DEV))
    prefill_backbone(m, h)
    plain = m._rt.x_bb.clone()
    m.drop_prefill_weights()
    prefill_backbone(m, h, a8=True)
    got = m._rt.x_bb.clone()
    kc = [b.kc.clone() for b in m.backbone.blocks]
    assert all(lin.f16 is None for b in m.backbone.blocks for lin in (b.qkv, b.o, b.w13, b.w2))
    x = h.reshape(B * P, -1).contiguous()
    pos = torch.arange(P, device=DEV).repeat(B)
    for i, b in enumerate(m.backbone.blocks):
        qkv = K.int8_mm_a8(K.rms(x, b.n1), b.qkv.q8, b.qkv.s8)
        q = torch.empty(B * P, b.h * b.hd, device=DEV).half()
        K.rope_cache(qkv, m.backbone.rope, pos, q, b.kc, b.vc, P, b.h, b.kvh, L)
        assert torch.equal(b.kc, kc[i])
        x = K.int8_mm_a8(K.prefill_attn(q, b.kc, b.vc, P), b.o.q8, b.o.s8, x)
        mm = K.int8_mm_a8(K.rms(x, b.n2), b.w13.q8, b.w13.s8, silu=True)
        x = K.int8_mm_a8(mm, b.w2.q8, b.w2.s8, x)
    assert torch.equal(got, x.view(B, P, -1)[:, -1])
    # a step of 1/127 of the largest activation: well inside a tenth of the state's norm
    assert float((got.float() - plain.float()).norm() / plain.float().norm()) < 0.1
    m.prompt_a8 = True
    ids = m.generate_ids(torch.randint(0, 1024, (P,)), 4, max_ms=320, seed=0, n=2)
    assert len(ids) == 2 and all(x.shape[0] == 8 for x in ids)


def test_registered_operators():
    """torch.ops.heartmula_b200.* equal the functions of the same name."""
    import estudiocanciones_b200.ops  # noqa: F401
    from estudiocanciones_b200 import kernels as K
    from estudiocanciones_b200.pages import PagePool
    ops = torch.ops.heartmula_b200
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5, 128, generator=g).half().to(DEV)
    w = torch.randint(-127, 128, (64, 128), generator=g, dtype=torch.int8).to(DEV)
    s = torch.full((64,), 0.01).half().to(DEV)
    q, sx = ops.quant_tokens(x)
    assert torch.equal(q, K.quant_tokens(x)[0]) and torch.equal(sx, K.quant_tokens(x)[1])
    assert torch.equal(ops.gemm_i8a8(q, sx, w, s), K.gemm_i8a8(q, sx, w, s))
    assert torch.equal(ops.int8_mm_a8(x, w, s, silu=True), K.int8_mm_a8(x, w, s, silu=True))
    ids = [torch.tensor(v, dtype=torch.int32, device=DEV) for v in ([0], [1], [2])]
    pools = []
    for o in (K, ops):
        p = PagePool(1, 12, 1, 64, 4, 64, 16, torch.float16, DEV)
        k, v = p.layer(0)
        o.pages_grow(p.table, p.lens, p.refs, 16, ids[0], 20)
        qkv = torch.randn(20, 3 * 64, generator=torch.Generator().manual_seed(1)).half().to(DEV)
        qo = torch.empty(20, 64, device=DEV).half()
        pos = torch.arange(20, device=DEV)
        rope = torch.randn(32, 32, 2, generator=torch.Generator().manual_seed(2)).to(DEV)
        o.rope_pages(qkv, rope, pos, qo, k, v, p.table, 20, 1, 1)
        o.pages_fork(p.k, p.v, p.table, p.lens, p.refs, ids[0], ids[1])
        o.pages_free(p.table, p.lens, p.refs, ids[0])
        n = o.pages_compact(p.k, p.v, p.table, p.refs)
        o.pages_copy(p.k, p.v, ids[0] * 0 + 1, ids[0] * 0 + 5)
        y = o.prefix_attn(qo[-1:], k, v, p.table, pos[-1:], seqs=ids[1])
        pools.append((p.k, p.v, p.table, p.lens, p.refs, n, qo, y))
    for a, b in zip(*pools):
        assert torch.equal(a, b)
    assert math.isfinite(float(pools[0][-1].float().sum()))
