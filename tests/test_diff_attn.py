"""Differential attention against its 64-bit form: every kernel over its head layouts, types, page sizes, lengths and masks; rows
that see no key, garbage in the places nobody sees, split passes, per-row lambda; the append and the attention run together as a
serving loop runs them; refusals."""
import numpy as np
import pytest
import torch

from espetero_b200 import capi, host, workloads as wl

from .diff_ref import U16, call_checks, diff64  # noqa: F401 (a fixture)

gpu = pytest.mark.gpu
EPS, SCALE = 1e-5, 0.6


def _weights(w, seed, per_row=False):
    rng = np.random.default_rng(seed)
    lam = rng.uniform(0.1, 0.9, size=(w.n_rows, w.H) if per_row else w.H).astype(np.float32)
    return lam, (1 + 0.2 * rng.standard_normal(w.HD)).astype(np.float32)


def _launch(w, lam, norm_w, options=None, tile_rows=None, plan_opts=None, stream=None, lam_ld=0, scratch=True, kv=None):
    """Plan, upload, run; (O bits, kernel)."""
    auto_rows, opts = host.diff_plan_options(w.trees, w.H, w.Hkv, w.HD)
    if tile_rows is not None:
        opts.update(tile_rows=tile_rows)
    opts.update(plan_opts or {})
    rows = opts["tile_rows"]
    op = host.AttnOp.for_workload(w, rows)
    try:
        for k, v in (options or {}).items():
            op.set_option(k, v)
        plan = host.plan_tiles(w.trees, w.Hkv, **opts)
        dp = op.upload(w)
        dev = op.device
        t = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)
        O = torch.full((w.n_rows, w.q_ld), 0x1234, dtype=torch.int16, device=dev)
        call = op.diff_call(plan, w.trees, dp.Q, dp.Kb, dp.Vb, O, kv=dp.kv, kv_scales=dp.kv_scales, blocks=dp.blocks, n_blocks=w.n_blocks, desc=dp.desc,
                            anc_mask=dp.anc_mask, lam=t(lam), lam_ld=lam_ld, norm_w=t(norm_w), eps=EPS, out_scale=SCALE, kv_base=w.kv_base,
                            scratch=None if scratch else torch.empty(0, dtype=torch.uint8, device=dev))
        if call.keep[5] is not None:
            call.keep[5].fill_(float("nan"))  # records must all be written before they are read
        torch.cuda.synchronize()
        op.diff_forward(call, stream)
        torch.cuda.synchronize()
        op.check_status()
        return O.cpu().numpy().view(np.uint16), op.last_kernel
    finally:
        op.close()


def _check(w, kernel=None, seed=3, norm=True, per_row=False, rounded=None, ref=None, **kw):
    lam, norm_w = _weights(w, seed, per_row)
    norm_w = norm_w if norm else None
    O, ran = _launch(w, lam, norm_w, lam_ld=w.H if per_row else 0, **kw)
    assert kernel is None or ran == kernel, ran
    # half a step of the softmax weights' type: none in diff_general; fp16 over E4M3 pools in diff_decode, else the pass's type
    unit = 0.0 if ran == "diff_general" else (2.0 ** -11 if (ran == "diff_decode" and w.kv_dtype == wl.E4M3) else U16[w.q_dtype])
    O64, tol = diff64(w, lam, norm_w, EPS, SCALE, unit)
    got = wl.from_bits16(O, w.q_dtype).astype(np.float64)
    bad = ~(np.abs(got - O64) <= tol)
    assert not bad.any(), f"{ran}: {int(bad.sum())} of {bad.size} off, worst {np.nanmax(np.abs(got - O64) / tol):.2f} of the bound, first at {np.argwhere(bad)[0]}"
    return O, ran


GENERAL = dict(attn_gqa=0, attn_umma=0)
# name, trees (P, M), H, Hkv, HD, bt, q type, pool, mask
GENERAL_CASES = [
    ("decode", [(0, 1), (1, 1), (77, 1), (400, 1)], 8, 2, 128, 16, wl.BF16, None, "causal"),
    ("odd pages", [(53, 1), (100, 9)], 4, 4, 64, 7, wl.F16, None, "causal"),
    ("512 dims", [(40, 3), (0, 33)], 2, 1, 512, 16, wl.BF16, None, "causal"),
    ("e4m3", [(130, 5), (1, 1)], 16, 2, 256, 32, wl.F16, wl.E4M3, "causal"),
    ("tree", [(90, 12), (0, 64)], 6, 2, 128, 16, wl.BF16, None, "tree"),
    ("forest", [(33, 40), (0, 17)], 4, 2, 64, 16, wl.F16, wl.E4M3, "forest"),
    ("groups of 9", [(65, 2)], 9, 1, 128, 16, wl.BF16, None, "causal"),
]


@gpu
@pytest.mark.parametrize("case", GENERAL_CASES, ids=[c[0] for c in GENERAL_CASES])
@pytest.mark.parametrize("split", [0, 32], ids=["whole", "split"])
def test_general(case, split):
    name, trees, H, Hkv, HD, bt, dt, pool, mask = case
    w = wl.make_pass(name, len(name), trees, H, Hkv, HD, bt, dt, pool, scale=(HD // 2) ** -0.5, mask=mask)
    _check(w, "diff_general", options=GENERAL, tile_rows=8, plan_opts=dict(split=split, groups=4096 if split else 1))


LENGTHS = [0, 1, 15, 16, 17, 31, 64, 65, 333, 1024]


@gpu
@pytest.mark.parametrize("HD", [128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (4, 2), (3, 1), (8, 2), (5, 1), (16, 2)], ids=lambda x: "H%d/%d" % x)
@pytest.mark.parametrize("types", [(wl.F16, None), (wl.BF16, None), (wl.F16, wl.E4M3), (wl.BF16, wl.E4M3)], ids=["f16", "bf16", "f16-e4m3", "bf16-e4m3"])
@pytest.mark.parametrize("split", [0, 32], ids=["whole", "split"])
def test_decode(HD, heads, types, split):
    w = wl.make_pass("decode", HD + heads[0], [(n, 1) for n in LENGTHS], heads[0], heads[1], HD, 48 if split else 16, types[0], types[1], scale=(HD // 2) ** -0.5)
    _check(w, "diff_decode", plan_opts=dict(split=split, groups=4096 if split else 1))


@gpu
def test_decode_long_and_hidden_from_itself():
    w = wl.make_pass("long", 3, [(40000, 1), (9, 1)], 8, 2, 128, 16, wl.BF16, scale=0.125)
    _check(w, "diff_decode")
    w = wl.make_pass("hidden", 3, [(100, 1), (0, 1), (0, 1)], 8, 2, 128, 16, wl.BF16, scale=0.125, mask="tree")
    w.anc_mask[:2] = 0
    O, _ = _check(w, "diff_decode")
    assert O[0].any() and not O[1].any() and O[2].any()


TC = {128: "diff_umma", 256: "diff_umma"}
# name, trees (P, M), H, Hkv, bt, pool, mask, tile_rows, split
ROWS_CASES = [
    ("prefill", [(0, 1), (0, 15), (0, 128), (0, 129), (0, 300)], 4, 2, 16, None, "causal", 128, 0),
    ("one head", [(0, 257)], 1, 1, 16, None, "causal", 128, 0),
    ("chunk", [(48, 130), (500, 77), (129, 1), (0, 64)], 8, 2, 32, None, "causal", 128, 0),
    ("chunk split", [(1000, 130), (500, 77)], 8, 2, 16, None, "causal", 128, 128),
    ("tree", [(300, 16), (0, 64), (17, 33)], 16, 2, 16, None, "tree", 16, 0),
    ("tree split", [(1030, 16), (600, 12), (64, 3)], 16, 2, 16, None, "tree", 16, 96),
    ("tree of 4 heads", [(260, 40)], 12, 3, 48, None, "tree", 32, 0),
    ("tree of 2 heads", [(260, 64), (0, 5)], 4, 2, 16, None, "tree", 64, 64),
    ("forest", [(100, 400), (0, 261)], 4, 2, 16, None, "forest", 128, 0),
    ("e4m3 chunk", [(333, 140), (16, 9)], 8, 2, 16, wl.E4M3, "causal", 128, 0),
    ("e4m3 tree split", [(700, 16), (90, 7)], 8, 1, 16, wl.E4M3, "tree", 16, 64),
    ("e4m3 prefill", [(0, 140)], 8, 2, 16, wl.E4M3, "causal", 128, 0),
]


@gpu
@pytest.mark.parametrize("HD", sorted(TC))
@pytest.mark.parametrize("dt", [wl.F16, wl.BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("case", ROWS_CASES, ids=[c[0] for c in ROWS_CASES])
def test_rows_on_tensor_cores(case, dt, HD):
    name, trees, H, Hkv, bt, pool, mask, tile_rows, split = case
    w = wl.make_pass(name, len(name) + HD, trees, H, Hkv, HD, bt, dt, pool, scale=(HD // 2) ** -0.5, mask=mask)
    _check(w, TC[HD], tile_rows=tile_rows, plan_opts=dict(split=split, groups=4096 if split else 1))


@gpu
@pytest.mark.parametrize("HD", sorted(TC))
def test_rows_over_e4m3_without_scratch(HD):
    w = wl.make_pass("no scratch", 4, [(64, 9)], 8, 2, HD, 16, wl.BF16, wl.E4M3, scale=0.125)
    _check(w, "diff_general", tile_rows=128, plan_opts=dict(split=0), scratch=False)


@gpu
@pytest.mark.parametrize("HD", [128, 256])
@pytest.mark.parametrize("shape", ["decode", "rows", "rows split"])
@pytest.mark.parametrize("order", ["rising", "falling", "wild"])
def test_page_scales_of_every_size(shape, order, HD):
    """V scales from 2^-24 to 2^6 within a sequence: the weights carry them, and neither end may leave fp16's range. Values
    small enough that products with the scales stay in the output's range."""
    trees = [(700, 1), (64, 1)] if shape == "decode" else [(700, 40), (64, 3)]
    w = wl.make_pass("scales", 4, trees, 8, 2, HD, 16, wl.F16, wl.E4M3, scale=(HD // 2) ** -0.5)
    n = 44
    e = np.linspace(-24, 6, n)
    e = {"rising": e, "falling": e[::-1], "wild": np.random.default_rng(3).permutation(e)}[order]
    for i, b in enumerate(w.blocks[:n]):
        w.kv_scales[b, 1] = 2.0 ** e[i]
    _check(w, None if shape == "decode" else TC.get(HD), tile_rows=8 if shape == "decode" else 128, plan_opts=dict(split=256 if shape == "rows split" else 0))


@gpu
@pytest.mark.parametrize("HD", sorted(TC))
def test_rows_with_scores_that_grow(HD):
    """Rows whose maximum rises by more than 2^8 from block to block: the accumulators are rescaled."""
    w = wl.make_pass("growing", 4, [(0, 600)], 2, 1, HD, 16, wl.F16, scale=(HD // 2) ** -0.5)
    K = wl.from_bits16(w.Kb, wl.F16) * (0.05 + np.arange(600)[:, None] / 60.0).astype(np.float32)
    w.Kb = wl.to_bits16(K.astype(np.float32), wl.F16)
    _check(w, TC[HD], tile_rows=128)


@gpu
@pytest.mark.parametrize("HD", sorted(TC))
def test_mixed_rows_in_one_pass(HD):
    """Single tokens beside a prompt and a chunk: one plan, one kernel."""
    w = wl.make_pass("mixed", 4, [(333, 1), (0, 200), (1, 1), (64, 30), (0, 1)], 8, 4, HD, 16, wl.BF16, scale=(HD // 2) ** -0.5)
    _check(w, TC[HD])


@gpu
@pytest.mark.parametrize("HD", sorted(TC))
def test_rows_report_a_block_outside_the_pool(HD):
    w = wl.make_pass("bad page", 3, [(300, 20)], 8, 2, HD, 16, wl.BF16, scale=0.125)
    for bad in (-1, w.n_blocks, 2 ** 30):
        w.blocks[2] = bad
        with pytest.raises(capi.EspError, match="bad block id"):
            _launch(w, *_weights(w, 1), tile_rows=128)


@gpu
@pytest.mark.parametrize("pool", [None, wl.E4M3], ids=["16-bit", "e4m3"])
def test_decode_reports_a_block_outside_the_pool(pool):
    """The page table's contents are seen by no host check: the kernel reads a block that exists instead and says so."""
    for options in (None, GENERAL):
        w = wl.make_pass("bad page", 3, [(100, 1), (50, 1)], 8, 2, 128, 16, wl.BF16, pool, scale=0.125)
        for bad in (-1, w.n_blocks, 2 ** 30):
            w.blocks[2] = bad
            with pytest.raises(capi.EspError, match="bad block id"):
                _launch(w, *_weights(w, 1), options=options)


@gpu
def test_no_norm_per_row_lambda_and_norm_of_nothing():
    w = wl.make_pass("plain", 5, [(70, 4), (0, 1)], 8, 2, 128, 16, wl.BF16, scale=0.125)
    _check(w, norm=False)
    _check(w, per_row=True)
    _check(w, per_row=True, options=GENERAL)


@gpu
def test_launches_on_the_stream_it_is_given():
    w = wl.make_pass("stream", 6, [(300, 1), (64, 1)], 8, 2, 128, 16, wl.F16, scale=0.125)
    lam, nw = _weights(w, 1)
    a, _ = _launch(w, lam, nw)
    b, _ = _launch(w, lam, nw, stream=torch.cuda.Stream().cuda_stream)
    assert np.array_equal(a, b)


@gpu
@pytest.mark.parametrize("options", [None, GENERAL], ids=["chosen", "general"])
def test_rows_that_see_nothing(options):
    """Ancestor masks of zero (padding nodes) without a cached key: zeros, with eps = 0 too; their neighbours are not disturbed."""
    w = wl.make_pass("empty rows", 7, [(0, 16), (64, 16)], 8, 2, 128, 16, wl.BF16, scale=0.125, mask="tree")
    w.anc_mask[[3, 15]] = 0
    w.anc_mask[[20]] = 0       # sees the 64 cached keys
    O, _ = _check(w, options=options, tile_rows=16, plan_opts=dict(split=0))
    assert not O[[3, 15]].any() and O[20].any()


@gpu
@pytest.mark.parametrize("options", [None, GENERAL], ids=["chosen", "general"])
@pytest.mark.parametrize("shape", ["decode", "rows"])
@pytest.mark.parametrize("HD", [128, 256])
def test_garbage_nobody_sees(options, shape, HD):
    """NaN and infinities in pool rows past P, in spare blocks and in batch rows behind the last tree."""
    trees = [(37, 1), (16, 1), (3, 1)] if shape == "decode" else [(37, 5), (0, 130), (250, 3)]
    w = wl.make_pass("garbage", 8, trees, 8, 2, HD, 16, wl.BF16, scale=0.125)
    rng = np.random.default_rng(0)
    pool = w.kv.reshape(w.n_blocks, 2, w.bt, w.kv_ld)
    live = np.zeros((w.n_blocks, w.bt), dtype=bool)
    for t in w.trees:
        j = np.arange(int(t["P"]))
        live[w.blocks[int(t["table"]) + j // w.bt], j % w.bt] = True
    for which in (0, 1):
        pool[:, which][~live] = rng.choice(np.array([0x7FC0, 0x7F80, 0xFF80], dtype=np.uint16), size=(int((~live).sum()), w.kv_ld))
    # rows behind the last tree: a padded batch
    pad = np.full((9, w.kv_ld), 0x7FC0, dtype=np.uint16)
    n = w.n_rows
    w.Kb, w.Vb = np.concatenate([w.Kb, pad]), np.concatenate([w.Vb, pad])
    w.Q = np.concatenate([w.Q, np.full((9, w.q_ld), 0x7FC0, dtype=np.uint16)])
    w.desc = np.concatenate([w.desc, np.zeros((9, 4), dtype=np.int32)])
    w.n_rows = n + 9
    lam, nw = _weights(w, 2)
    O, ran = _launch(w, lam, nw, options=options)
    assert (O[n:] == 0x1234).all()  # rows of no tree stay as they were
    O64, tol = diff64(w, lam, nw, EPS, SCALE, 0.0 if ran == "diff_general" else U16[w.q_dtype])
    got = wl.from_bits16(O[:n], w.q_dtype).astype(np.float64)
    assert (np.abs(got - O64[:n]) <= tol[:n]).all()


@gpu
def test_same_bits_every_time():
    w = wl.make_pass("repeat", 9, [(5000, 1), (900, 1)], 32, 4, 128, 16, wl.BF16, scale=0.125)
    lam, nw = _weights(w, 4)
    runs = [_launch(w, lam, nw)[0] for _ in range(3)]
    assert np.array_equal(runs[0], runs[1]) and np.array_equal(runs[0], runs[2])


@gpu
@pytest.mark.parametrize("pool", [None, wl.E4M3], ids=["16-bit", "e4m3"])
def test_a_serving_loop(pool):
    """A prompt, then tokens one by one: kv_append writes the cache that diff_forward reads, in one captured step after another.
    The last token's output is what one pass over the whole sequence gives."""
    H, Hkv, HD, bt, n, steps = 8, 2, 128, 16, 45, 6
    dev = torch.device("cuda", 0)
    rng = np.random.default_rng(12)
    total = n + steps
    X = torch.from_numpy(rng.standard_normal((total, (H + 2 * Hkv) * HD)).astype(np.float32)).to(dev).to(torch.float16)
    n_blocks = (total + bt - 1) // bt + 1
    blocks = torch.from_numpy(rng.permutation(n_blocks).astype(np.int32)).to(dev)
    slots = torch.stack([blocks[torch.arange(total, device=dev) // bt], (torch.arange(total, device=dev) % bt).int()], dim=1).int().contiguous()
    inv = torch.from_numpy((1e4 ** (-np.arange(32) / 32)).astype(np.float32)).to(dev)
    pos = torch.arange(total, dtype=torch.int32, device=dev)
    kv_dtype = wl.F16 if pool is None else pool
    kv = torch.zeros(n_blocks * 2 * bt * Hkv * HD, dtype=torch.int16 if pool is None else torch.uint8, device=dev)
    scales = None if pool is None else torch.full((n_blocks, 2, Hkv), 2.0 ** -6, device=dev)
    lam = torch.full((H,), 0.4, device=dev)
    nw = torch.ones(HD, device=dev)

    def step(at, rows, keep):
        trees = host.make_trees([rows], [at], [0])
        tr, opts = host.diff_plan_options(trees, H, Hkv, HD)
        op = host.AttnOp(H, Hkv, HD, bt, wl.F16, kv_dtype, 0.125, 0, tr)
        q, k, v = X[at:at + rows].split([H * HD, Hkv * HD, Hkv * HD], dim=1)
        Q, O = (torch.zeros((rows, H * HD), dtype=torch.float16, device=dev) for _ in range(2))
        Kb, Vb = (torch.zeros((rows, Hkv * HD), dtype=torch.float16, device=dev) for _ in range(2))
        app = op.append_call(q, k, v, Q, Kb, Vb, kv=kv, kv_scales=scales, n_blocks=n_blocks, slots=slots[at:at + rows], pos=pos[at:at + rows], inv_freq=inv, maps=2)
        desc = torch.zeros((rows, 4), dtype=torch.int32, device=dev)
        att = op.diff_call(host.plan_tiles(trees, Hkv, **opts), trees, Q, Kb, Vb, O, kv=kv, kv_scales=scales, blocks=blocks, n_blocks=n_blocks, desc=desc, lam=lam,
                           norm_w=nw, eps=EPS, out_scale=SCALE)
        op.kv_append(app)
        op.diff_forward(att)
        want = O.clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()  # the same step captured and replayed gives the same
        with torch.cuda.graph(g):
            op.kv_append(app)
            op.diff_forward(att)
        O.zero_()
        g.replay()
        g.replay()
        torch.cuda.synchronize()
        op.check_status()
        assert torch.equal(O, want)
        keep.append((op, app, att, Q, Kb, Vb))
        return O

    keep = []
    step(0, n, keep)
    for i in range(steps):
        last = step(n + i, 1, keep)
    Q, Kb, Vb = (torch.cat([k[j] for k in keep]) for j in (3, 4, 5))
    w = wl.make_pass("whole", 1, [(0, total)], H, Hkv, HD, bt, wl.F16, scale=0.125)
    bits = lambda t: t.cpu().view(torch.int16).numpy().view(np.uint16)
    w.Q, w.Kb, w.Vb = bits(Q), bits(Kb), bits(Vb)
    if pool is not None:  # what the cache holds of them
        for x in (w.Kb, w.Vb):
            x[:total - 1] = wl.to_bits16(wl.e4m3_decode(wl.e4m3_encode(wl.from_bits16(x[:total - 1], wl.F16) * 64.0)) / 64.0, wl.F16)
    O64, tol = diff64(w, np.full(H, 0.4, dtype=np.float32), np.ones(HD, dtype=np.float32), EPS, SCALE, U16[wl.F16])
    assert (np.abs(last.cpu().numpy().astype(np.float64) - O64[-1:]) <= tol[-1:]).all()
    for k in keep:
        k[0].close()


@gpu
@pytest.mark.parametrize("HD", [128, 256])
def test_a_pass_again_and_replayed(HD):
    """Split passes, one after another on one context and in a replayed graph, all give the first one's bits."""
    w = wl.make_pass("again", 9, [(1000, 1), (130, 1), (700, 1)], 8, 2, HD, 16, wl.BF16, scale=0.125)
    lam, nw = _weights(w, 4)
    op = host.AttnOp.for_workload(w, 8)
    dp = op.upload(w)
    plan = host.plan_tiles(w.trees, w.Hkv, **dict(host.diff_plan_options(w.trees, w.H, w.Hkv, HD)[1], groups=40))
    assert 1 < max(plan.jobs["nparts"]) <= 16
    O = torch.zeros((w.n_rows, w.q_ld), dtype=torch.int16, device=op.device)
    call = op.diff_call(plan, w.trees, dp.Q, dp.Kb, dp.Vb, O, kv=dp.kv, blocks=dp.blocks, n_blocks=w.n_blocks, desc=dp.desc, lam=torch.from_numpy(lam).cuda(),
                        norm_w=torch.from_numpy(nw).cuda(), eps=EPS, out_scale=SCALE)
    before = op.launch_count
    op.diff_forward(call)
    torch.cuda.synchronize()
    assert op.launch_count == before + 2
    want = O.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.diff_forward(call)
    for _ in range(5):
        O.zero_()
        call.keep[5].fill_(float("nan"))
        op.diff_forward(call)
        torch.cuda.synchronize()
        assert torch.equal(O, want)
        O.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(O, want)
    op.check_status()
    op.close()


@gpu
@pytest.mark.parametrize("options", [None, GENERAL], ids=["chosen", "general"])
@pytest.mark.parametrize("shape", ["decode", "rows"])
@pytest.mark.parametrize("pool", [None, wl.E4M3], ids=["16-bit", "e4m3"])
def test_a_padded_block_table(pool, shape, options):
    """Table entries that no tile reads may hold anything, NaN codes behind P are never mixed in."""
    w = wl.make_pass("padded", 12, [(37, 1), (250, 1)] if shape == "decode" else [(37, 5), (250, 3)], 8, 2, 128, 16, wl.F16, pool, scale=0.125)
    w.blocks = np.concatenate([w.blocks, np.array([-1, -7, w.n_blocks, 2 ** 30, -1], dtype=np.int32)])
    if pool == wl.E4M3:
        kv = w.kv.reshape(w.n_blocks, 2, w.bt, w.kv_ld)
        for t in w.trees:
            kv[w.blocks[int(t["table"]) + int(t["P"]) // w.bt], :, int(t["P"]) % w.bt:] = 0x7F
    _check(w, options=options)


@gpu
def test_check_finite_scans_these_passes():
    w = wl.make_pass("finite", 13, [(200, 1), (100, 1)], 8, 2, 128, 16, wl.BF16, scale=0.125)
    w.kv.reshape(w.n_blocks, 2, w.bt, w.kv_ld)[int(w.blocks[int(w.trees[1]["table"])]), 1, 3, 5] = 0x7FC0
    lam, nw = _weights(w, 1)
    _launch(w, lam, nw)
    with pytest.raises(capi.EspError, match="row 1, column 0"):  # the norm carries it into the whole head
        _launch(w, lam, nw, options=dict(check_finite=1))


@gpu
def test_two_passes_of_one_context_at_once():
    """Split passes that share a context, eagerly on two streams and as two graphs: each gives the bits it gives alone."""
    ws = [wl.make_pass("left", 14, [(3000, 40)], 8, 2, 128, 16, wl.F16, wl.E4M3, scale=0.125), wl.make_pass("right", 15, [(2500, 24), (40, 3)], 8, 2, 128, 16, wl.F16, wl.E4M3, scale=0.125)]
    op = host.AttnOp.for_workload(ws[0], 32)
    calls, outs, want = [], [], []
    for i, w in enumerate(ws):
        lam, nw = _weights(w, i)
        dp = op.upload(w)
        O = torch.zeros((w.n_rows, w.q_ld), dtype=torch.int16, device=op.device)
        plan = host.plan_tiles(w.trees, w.Hkv, **dict(host.diff_plan_options(w.trees, w.H, w.Hkv, w.HD, w.kv_dtype)[1], tile_rows=32, split=300, groups=64))
        assert plan.n_parts
        calls.append(op.diff_call(plan, w.trees, dp.Q, dp.Kb, dp.Vb, O, kv=dp.kv, kv_scales=dp.kv_scales, blocks=dp.blocks, n_blocks=w.n_blocks, desc=dp.desc,
                                  lam=torch.from_numpy(lam).cuda(), norm_w=torch.from_numpy(nw).cuda(), eps=EPS, out_scale=SCALE))
        op.diff_forward(calls[i])
        torch.cuda.synchronize()
        outs.append(O), want.append(O.clone())
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs = []
    for c in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            op.diff_forward(c)
    for turn in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for _ in range(5):
            for s, c, g in zip(streams, calls, graphs):
                with torch.cuda.stream(s):
                    g.replay() if turn % 2 else op.diff_forward(c)
        torch.cuda.synchronize()
        for o, x in zip(outs, want):
            assert torch.equal(o, x)
    op.check_status()
    op.close()


@gpu
def test_rows_with_other_strides_are_refused():
    w = wl.make_pass("strides", 16, [(0, 4)], 8, 2, 128, 16, wl.F16, scale=0.125)
    op = host.AttnOp.for_workload(w, 8)
    dp = op.upload(w)
    plan = host.plan_tiles(w.trees, w.Hkv)
    wide = torch.zeros((4, 2 * w.q_ld), dtype=torch.int16, device=op.device)
    good = dict(Q=dp.Q, Kb=dp.Kb, Vb=dp.Vb, O=torch.zeros_like(dp.Q), desc=dp.desc, lam=torch.zeros(8, device=op.device))
    for name, t in (("Kb", wide[:, :w.kv_ld]), ("Vb", wide[:, :w.kv_ld]), ("O", wide[:, :w.q_ld]), ("Q", wide[:, ::2])):
        with pytest.raises(ValueError, match=name):
            op.diff_call(plan, w.trees, **dict(good, **{name: t}))
    for name, t in (("Kb", wide[:, :w.kv_ld]), ("K", wide[:, :2 * w.kv_ld:2])):
        with pytest.raises(ValueError, match=name):
            op.append_call(**dict(dict(Q=dp.Q, K=dp.Kb, V=dp.Vb, Qo=dp.Q, Kb=dp.Kb, Vb=dp.Vb), **{name: t}))
    op.close()


@gpu
@pytest.mark.parametrize("H,dim", [(1, 1), (32, 64), (7, 129)])
def test_lambda(H, dim):
    rng = np.random.default_rng(H)
    v = [(0.2 * rng.standard_normal((H, dim))).astype(np.float32) for _ in range(4)]
    op = host.AttnOp(8, 2, 128, 16, wl.BF16, wl.BF16, 1.0)
    t = [torch.from_numpy(x).cuda() for x in v]
    for vec, dev in ((v, t), ([x[:1] for x in v], [x[0] for x in t])):
        got = op.diff_lambda(*dev, lambda_init=0.3, H=H).cpu().numpy().astype(np.float64)
        a, b = (np.exp((vec[i].astype(np.float64) * vec[i + 1]).sum(axis=1)) for i in (0, 2))
        mag = sum((np.abs(vec[i].astype(np.float64) * vec[i + 1])).sum(axis=1) for i in (0, 2))
        # a dot of dim terms: dim 2^-24 of its magnitude; expf within 2 steps; two sums
        assert (np.abs(got - (a - b + 0.3)) <= (a + b) * (mag * (dim + 2) * 2.0 ** -24 + 6 * 2.0 ** -24) + 2.0 ** -23).all()
    op.close()


# ---------------------------------------------------------------------------------------------- without a GPU
def test_plan_options():
    """Options suit the pass: single rows are cut for the whole GPU, passes over their own rows are not cut at all."""
    tr, o = host.diff_plan_options(host.make_trees([1, 1], [5000, 1], [0, 313]), 32, 4, 128)
    assert tr == 8 and o["split"] > 0
    tr, o = host.diff_plan_options(host.make_trees([700], [0], [0]), 32, 4, 128)
    assert tr == 128 and len(host.plan_tiles(host.make_trees([700], [0], [0]), 4, **o).jobs) == 0
    for H, Hkv, rows in ((32, 4, 16), (8, 8, 128), (24, 4, 64), (16, 8, 64)):
        tr, o = host.diff_plan_options(host.make_trees([16] * 4, [4096] * 4, [0] * 4), H, Hkv, 128)
        assert tr == rows == o["tile_rows"]


def test_plan_options_and_lambda_refuse_bad_arguments():
    lib = capi.load()
    o = capi.PlanOpts()
    assert lib.esp_diff_plan_opts(None, None, 0, o) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_plan_opts(capi.Shape(7, 2, 128), None, 0, o) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_plan_opts(capi.Shape(8, 2, 128), None, 3, o) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_plan_opts(capi.Shape(8, 2, 128), None, 0, o) == 0
    assert lib.esp_diff_forward(None, None, capi.Args(), capi.DiffArgs()) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_lambda(None, None, None, None, None, 4, 64, 0, 0.1, None) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_lambda(None, None, None, None, None, 4, 0, 0, 0.1, None) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_lambda(None, None, None, None, None, 4, 64, 63, 0.1, None) == capi.ESP_ERR_INVALID
    assert lib.esp_diff_lambda(None, None, None, None, None, 0, 64, 0, 0.1, None) == 0
    s = capi.Shape(32, 8, 256, 16, capi.ESP_BF16, capi.ESP_E4M3, 8, 0, 0.0625)
    assert lib.esp_diff_parts_floats(s, 32) == 2 * lib.esp_attn_parts_floats(s, 32)


def test_forward_refuses_bad_arguments(call_checks):  # noqa: F811
    import ctypes as C
    trees = host.make_trees([4, 1], [20, 3], [0, 2])
    plan = host.plan_tiles(trees, 2)
    keep = []

    def code(flags=0, diff=None, tiles=None, **more):
        shape = capi.Shape(8, 2, 128, 16, wl.BF16, wl.BF16, 8, flags, 0.125)
        t = plan.tiles.copy()
        for k, v in (tiles or {}).items():
            t[k][0] = v
        keep.append(t)
        a = capi.Args(Q=0x10000, Kb=0x20000, Vb=0x30000, kv=0x40000, blocks=0x50000, desc=0x60000, O=0x70000, tiles=0x80000, trees=0x90000,
                      tiles_host=t.ctypes.data, trees_host=trees.ctypes.data, n_tiles=len(t), n_trees=2, n_rows=5, n_blocks=9, n_block_entries=3)
        a.p = capi.Params(8, 2, 1024, 256, 2048, 16, 0)
        for k, v in more.items():
            setattr(a, k, v)
        d = capi.DiffArgs(0x100000, 0x110000, 0, 1e-5, 1.0)
        for k, v in (diff or {}).items():
            setattr(d, k, v)
        return call_checks.diff(shape, a, d)

    assert code() == 0
    assert code(diff=dict(norm_w=None)) == 0 and code(diff=dict(lam_ld=8)) == 0
    for more in (dict(window=5), dict(ring=2), dict(bidi=1), dict(qsa_tlist=0x1000), dict(flags=capi.ESP_ATTN_FLAG_GATE)):
        assert code(**more) == capi.ESP_ERR_UNSUPPORTED, more
    nan = float("nan")
    for more in (dict(lse=0x1000), dict(diff=dict(lam=None)), dict(diff=dict(lam_ld=7)), dict(diff=dict(lam_ld=-8)), dict(diff=dict(eps=-1.0)), dict(diff=dict(eps=nan)),
                 dict(diff=dict(out_scale=nan)), dict(diff=dict(norm_w=0x110008)), dict(Q=None), dict(O=0x70008), dict(desc=None), dict(n_rows=4), dict(n_block_entries=2),
                 dict(kv=None), dict(tiles=dict(tree=2)), dict(tiles=dict(k1=21)), dict(tiles=dict(k0=-1)), dict(tiles=dict(r0=4)), dict(tiles=dict(part=0)),
                 dict(flags=capi.ESP_ATTN_FLAG_ANC_MASK)):
        assert code(**more) == capi.ESP_ERR_INVALID, more
    assert C.sizeof(capi.DiffArgs) == 32
