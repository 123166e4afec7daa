"""Differential attention at the edges of what its documentation allows: mask records outside their tree, garbage in rows that nobody
sees, page scales and queries of every magnitude, layers behind the pool's first, wide row strides; and the plans and refusals that
go with them."""
import ctypes as C

import numpy as np
import pytest
import torch

from espetero_b200 import capi, host, workloads as wl

from .diff_ref import SUB16, U16, call_checks, diff64, keys_values, visible  # noqa: F401 (a fixture)

gpu = pytest.mark.gpu
EPS, SCALE = 1e-5, 0.6
GENERAL = dict(attn_gqa=0, attn_umma=0)


def _weights(w, seed):
    rng = np.random.default_rng(seed)
    return rng.uniform(0.1, 0.9, size=w.H).astype(np.float32), (1 + 0.2 * rng.standard_normal(w.HD)).astype(np.float32)


def _run(w, lam, norm_w, options=None, tile_rows=None, split=None, eps=EPS):
    """One pass as its plan options say, or in tiles of `tile_rows`; (O as float64, kernel)."""
    auto_rows, opts = host.diff_plan_options(w.trees, w.H, w.Hkv, w.HD, w.kv_dtype)
    opts.update(tile_rows=tile_rows or auto_rows)
    if split is not None:
        opts.update(split=split, groups=4096 if split else 1)
    op = host.AttnOp.for_workload(w, opts["tile_rows"])
    try:
        for k, v in (options or {}).items():
            op.set_option(k, v)
        dp = op.upload(w)
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(op.device)
        O = torch.full((w.n_rows, w.q_ld), 0x1234, dtype=torch.int16, device=op.device)
        call = op.diff_call(host.plan_tiles(w.trees, w.Hkv, **opts), w.trees, dp.Q, dp.Kb, dp.Vb, O, kv=dp.kv, kv_scales=dp.kv_scales, blocks=dp.blocks, n_blocks=w.n_blocks,
                            desc=dp.desc, anc_mask=dp.anc_mask, lam=t(lam), norm_w=t(norm_w), eps=eps, out_scale=SCALE, kv_base=w.kv_base)
        op.diff_forward(call)
        torch.cuda.synchronize()
        op.check_status()
        return wl.from_bits16(O.cpu().numpy().view(np.uint16), w.q_dtype).astype(np.float64), op.last_kernel
    finally:
        op.close()


def _unit(w, ran):
    """Half a step of the type that the softmax weights are rounded to."""
    return 0.0 if ran == "diff_general" else (2.0 ** -11 if (ran == "diff_decode" and w.kv_dtype == wl.E4M3) else U16[w.q_dtype])


def _check(w, kernel=None, seed=3, **kw):
    lam, norm_w = _weights(w, seed)
    got, ran = _run(w, lam, norm_w, **kw)
    assert kernel is None or ran == kernel, ran
    O64, tol = diff64(w, lam, norm_w, EPS, SCALE, _unit(w, ran))
    bad = ~(np.abs(got - O64) <= tol)
    assert not bad.any(), f"{ran}: {int(bad.sum())} of {bad.size} off, first at {np.argwhere(bad)[0]}"
    return got, ran


@gpu
@pytest.mark.parametrize("options", [None, GENERAL], ids=["chosen", "general"])
@pytest.mark.parametrize("HD", [128, 256])
def test_mask_records_outside_their_tree(options, HD):
    """desc records whose ancestor length is negative (none) or past the tree (all of it), and whose segment starts past the row (a row
    that sees nothing; in the third tree all of them) or before the tree. 300 and 200 rows end inside a block of 128 keys."""
    w = wl.make_pass("records", 21, [(0, 300), (40, 200), (0, 3)], 4, 2, HD, 16, wl.BF16, scale=(HD // 2) ** -0.5)
    far = 2 ** 31 - 1
    w.desc[:, 2] = -1000
    w.desc[260:, 0] = -far - 1
    w.desc[[5, 299, 310, 500, 501, 502], 0] = far
    w.desc[[130, 320], 2] = far
    w.desc[131, 2] = -far - 1
    got, _ = _check(w, None if options else "diff_umma", options=options, tile_rows=128, split=0)
    assert not got[[5, 299, 500, 501, 502]].any() and got[310].any()  # row 310 sees its 40 cached keys


@gpu
@pytest.mark.parametrize("options", [None, GENERAL], ids=["chosen", "general"])
@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("HD", [128, 256])
def test_garbage_in_tree_nodes_that_nobody_sees(options, tile_rows, HD):
    """Padding nodes: their mask is empty and in no other node's mask; their keys and values hold NaN and infinities."""
    w = wl.make_pass("padding nodes", 22, [(0, 16), (64, 40), (20, 64)], 8, 1, HD, 16, wl.BF16, scale=(HD // 2) ** -0.5, mask="tree")
    unseen = {0: [3, 15], 16: [0, 31, 32, 39], 56: [17, 63]}
    for base, nodes in unseen.items():
        rows = w.anc_mask[base:base + 64 if base == 56 else base + (16 if base == 0 else 40)]
        for j in nodes:
            rows &= ~np.uint64(1 << j)
            rows[j] = 0
            w.Kb[base + j], w.Vb[base + j] = 0x7FC0, np.resize(np.array([0x7FC0, 0x7F80, 0xFF80], dtype=np.uint16), w.kv_ld)
    got, _ = _check(w, None if options else "diff_umma", options=options, tile_rows=tile_rows, split=0)
    assert not got[[3, 15]].any() and got[[16, 55, 73]].any(axis=1).all()


def _uneven_pages(HD, rows, split, page, log2_scale, below, share):
    """An fp16 pass over E4M3 pages. One page's V scale is 2^log2_scale and its keys score `below` under the others', whose V scale is 2^-20; the pass's own
    keys score 60 below. Every weight has to keep its bits beside the others'. `share`: least and largest part that the page may have of a row.
    The bound: weights p_j s_j are rounded to half a step of fp16, or to half a subnormal step in units of at most twice the row's largest
    p_j s_j; a code is at most 448. The rest as in diff64."""
    w = wl.make_pass("uneven", 23, [(96, rows)], 8, 2, HD, 16, wl.F16, wl.E4M3, scale=1.0)
    d = HD // 2
    Q = np.full((rows, w.H, 2, d), 0.125, dtype=np.float32)
    w.Q = wl.to_bits16(Q.reshape(rows, -1), wl.F16)
    pool = w.kv.reshape(w.n_blocks, 2, w.bt, w.Hkv, HD)
    rng = np.random.default_rng(5)
    for i, b in enumerate(w.blocks):
        k = rng.uniform(-1.0, 1.0, size=(w.bt, w.Hkv, HD)) - (8.0 * below / d if i == page else 0.0)
        pool[b, 0] = wl.e4m3_encode((k * 8).astype(np.float32))
        w.kv_scales[b, 0], w.kv_scales[b, 1] = 0.125, 2.0 ** (log2_scale if i == page else -20)
    w.Kb = wl.to_bits16((rng.uniform(-1, 1, size=(rows, w.kv_ld)) - 480.0 / d).astype(np.float32), wl.F16)
    lam, norm_w = _weights(w, 3)
    eps = 1e-14
    got, ran = _run(w, lam, norm_w, tile_rows=8 if rows == 1 else 128, split=split, eps=eps)
    assert ran == ("diff_decode" if rows == 1 else "diff_umma")
    O64, _ = diff64(w, lam, norm_w, eps, SCALE, 0.0)
    unit, n = U16[wl.F16], 96 + rows
    for kvh in range(w.Hkv):
        K, V, _ = keys_values(w, 0, kvh)
        size = np.ones(n)  # the page's scale beside every key
        size[:96] = np.repeat(w.kv_scales[w.blocks, 1, kvh], w.bt)
        for h in range(kvh * 4, kvh * 4 + 4):
            D, e = 0.0, 0.0
            for c, f in ((0, 1.0), (1, float(lam[h]))):
                s = np.where(visible(w, 0), Q[:, h, c].astype(np.float64) @ K[:, c * d:(c + 1) * d].T, -np.inf)
                p = np.exp(s - s.max(axis=1, keepdims=True))
                p /= p.sum(axis=1, keepdims=True)
                part = (p * size)[:, 16 * page:16 * page + 16].sum(axis=1) / (p * size).sum(axis=1)
                assert (share[0] <= part).all() and (part <= share[1]).all()
                es = 0.125 * np.abs(K[:, c * d:(c + 1) * d]).sum(axis=1).max() * (d + 2) * 2.0 ** -24
                D = D + (f if c == 0 else -f) * (p @ V)
                e = e + f * ((2 * es + 2.0 ** -21 + (n + 8) * 2.0 ** -24 + unit) * (p @ np.abs(V)) + n * 448 * 2.0 ** -24 * (p * size).max(axis=1, keepdims=True))
            norm = np.sqrt((D * D).sum(axis=1, keepdims=True))
            fac = SCALE / np.sqrt((D * D).mean(axis=1, keepdims=True) + eps) * norm_w
            tol = 1.02 * np.abs(fac) * (e + np.abs(D) * np.sqrt((e * e).sum(axis=1, keepdims=True)) / norm) + (unit + 2.0 ** -20) * np.abs(fac * D) + SUB16[wl.F16]
            cols = slice(h * HD, (h + 1) * HD)
            assert np.allclose(O64[:, cols], fac * D, rtol=1e-9, atol=1e-12)
            err = np.abs(got[:, cols] - O64[:, cols])
            assert (err <= tol).all(), (ran, float((err / tol).max()), float(np.abs(got[:, cols]).max()))


@gpu
@pytest.mark.parametrize("split", [0, 32], ids=["whole", "split"])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("HD", [128, 256])
def test_a_page_of_large_values_that_is_hardly_attended(HD, rows, split):
    """Weights of e^-60 on values of 2^6, the first page's: the rows are what the small pages hold."""
    _uneven_pages(HD, rows, split, 0, 6, 60.0, (0.0, 1e-6))


@gpu
@pytest.mark.parametrize("split", [0, 32], ids=["whole", "split"])
@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("HD", [128, 256])
def test_a_page_of_large_values_that_carries_a_small_weight(HD, rows, split):
    """Weights of e^-17 on values of 2^10, the last page's: the rows are mostly what the large page holds."""
    _uneven_pages(HD, rows, split, 5, 10, 17.0, (0.7, 1.0))


@gpu
@pytest.mark.parametrize("power", [-40, 0, 30])
@pytest.mark.parametrize("heads", [(8, 2), (8, 1)], ids=["4 heads", "8 heads"])
@pytest.mark.parametrize("HD", [128, 256])
def test_queries_of_every_magnitude_over_e4m3(HD, heads, power):
    """bf16 queries far outside fp16's range, their keys as far the other way: the scores are ordinary. One head is all zeros."""
    w = wl.make_pass("magnitude", 24, [(100, 1), (33, 1), (0, 1)], heads[0], heads[1], HD, 16, wl.BF16, wl.E4M3, scale=(HD // 2) ** -0.5)
    f = np.float32(2.0 ** power)
    Q = wl.from_bits16(w.Q, wl.BF16) * f
    Q[0, :HD] = 0.0
    w.Q = wl.to_bits16(Q, wl.BF16)
    w.Kb = wl.to_bits16(wl.from_bits16(w.Kb, wl.BF16) / f, wl.BF16)
    w.kv_scales[:, 0] /= f
    _check(w, "diff_decode")


@gpu
@pytest.mark.parametrize("types", [(wl.F16, None), (wl.BF16, wl.E4M3)], ids=["f16", "bf16-e4m3"])
@pytest.mark.parametrize("heads", [(32, 2), (32, 1), (12, 1), (9, 1)], ids=lambda x: "H%d/%d" % x)
@pytest.mark.parametrize("HD", [128, 256])
def test_single_rows_of_many_heads(HD, heads, types):
    """More than 8 query heads to a kv head, as the options plan them: on the tensor cores."""
    w = wl.make_pass("many heads", 25, [(n, 1) for n in (0, 1, 15, 16, 17, 130, 333, 2000)], heads[0], heads[1], HD, 16, types[0], types[1], scale=(HD // 2) ** -0.5)
    _check(w, "diff_umma")


@gpu
@pytest.mark.parametrize("pool", [None, wl.E4M3], ids=["16-bit", "e4m3"])
@pytest.mark.parametrize("tile_rows", [None, 16])
def test_idle_slots_of_a_batch(pool, tile_rows):
    """Trees without rows beside single tokens: the same kernel as without them, and right."""
    w = wl.make_pass("idle", 26, [(0, 0), (300, 1), (50, 0), (1, 1), (0, 0), (64, 1), (9, 0)], 8, 2, 128, 16, wl.BF16, pool, scale=0.125)
    _check(w, "diff_decode", tile_rows=tile_rows)
    w = wl.make_pass("idle rows", 26, [(0, 0), (300, 20), (50, 0), (1, 1)], 8, 2, 128, 16, wl.BF16, pool, scale=0.125)
    _check(w, "diff_general" if tile_rows else "diff_umma", tile_rows=tile_rows)  # tiles of 16 rows want 8 heads to a kv head


@gpu
@pytest.mark.parametrize("heads", [(8, 2), (8, 1)], ids=["4 heads", "8 heads"])
@pytest.mark.parametrize("HD", [128, 256])
def test_e4m3_steps_as_they_are_planned(HD, heads):
    """Plans for the pool's own type: three or two CTAs to an SM, uneven lengths split for them."""
    w = wl.make_pass("planned", 27, [(n, 1) for n in (9000, 1, 2500, 0, 4097)], heads[0], heads[1], HD, 16, wl.BF16, wl.E4M3, scale=(HD // 2) ** -0.5)
    assert _planned([1] * 5, w.trees["P"], *heads, HD, wl.E4M3)[1] > 8
    _check(w, "diff_decode")


def _apart(w, entries, fill):
    """The same pass with `entries` table entries per tree, those that no tree reads set to `fill` (valid pages or not)."""
    blocks = np.resize(np.asarray(fill, dtype=np.int32), len(w.trees) * entries)
    for i, t in enumerate(w.trees):
        n = (int(t["P"]) + w.bt - 1) // w.bt
        blocks[i * entries:i * entries + n] = w.blocks[int(t["table"]):int(t["table"]) + n]
        t["table"] = i * entries
    w.blocks = blocks
    return w


@gpu
@pytest.mark.parametrize("HD", [128, 256])
def test_only_the_pages_that_are_read_are_widened(HD):
    """A table with room for many more pages than its sequences have: the scratch of the entries behind them is left as it was; their
    content may be anything, and what the trees read is right. Two trees share one table, one has no rows, one no cached keys."""
    w = wl.make_pass("padded", 28, [(300, 20), (50, 0), (1000, 33), (0, 9), (300, 5)], 8, 2, HD, 16, wl.F16, wl.E4M3, scale=(HD // 2) ** -0.5)
    w = _apart(w, 100, [0, -1, 3, w.n_blocks, 2 ** 30])
    w.trees[4]["table"] = w.trees[0]["table"]
    lam, norm_w = _weights(w, 3)
    op = host.AttnOp.for_workload(w, 32)
    dp = op.upload(w)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(op.device)
    O = torch.full((w.n_rows, w.q_ld), 0x1234, dtype=torch.int16, device=op.device)
    page = 2 * w.bt * w.kv_ld * 2
    scratch = torch.full((int(op.lib.esp_attn_dequant_scratch_bytes(C.byref(op.shape), len(w.blocks))),), 0xA5, dtype=torch.uint8, device=op.device)
    _, opts = host.diff_plan_options(w.trees, w.H, w.Hkv, w.HD, w.kv_dtype)
    call = op.diff_call(host.plan_tiles(w.trees, w.Hkv, **dict(opts, tile_rows=32)), w.trees, dp.Q, dp.Kb, dp.Vb, O, kv=dp.kv, kv_scales=dp.kv_scales, blocks=dp.blocks,
                        n_blocks=w.n_blocks, desc=dp.desc, lam=t(lam), norm_w=t(norm_w), eps=EPS, out_scale=SCALE, scratch=scratch)
    op.diff_forward(call)
    torch.cuda.synchronize()
    op.check_status()
    assert op.last_kernel == "diff_umma"
    O64, tol = diff64(w, lam, norm_w, EPS, SCALE, U16[wl.F16])
    assert (np.abs(wl.from_bits16(O.cpu().numpy().view(np.uint16), wl.F16).astype(np.float64) - O64) <= tol).all()
    pages = scratch[:len(w.blocks) * page].view(len(w.blocks), page)
    left = (pages == 0xA5).all(dim=1).cpu().numpy()
    read = np.zeros(len(w.blocks), dtype=bool)
    for tree in w.trees:
        if tree["M"]:
            read[int(tree["table"]):int(tree["table"]) + (int(tree["P"]) + 15) // 16] = True
    assert (left == ~read).all()
    op.close()


@gpu
@pytest.mark.parametrize("apart", [0, 20], ids=["tight", "padded"])
def test_many_trees_over_e4m3(apart):
    """More trees than a warp sums up at once, some without rows, some without cached keys, every seventh with its neighbour's table."""
    w = wl.make_pass("many", 31, [((37 * i) % 290, (0, 1, 2, 5)[i % 4]) for i in range(75)], 4, 2, 128, 16, wl.F16, wl.E4M3, scale=0.125)
    if apart:
        w = _apart(w, apart, [-1, 0, 2 ** 30])
    for i in range(7, 75, 7):
        w.trees[i]["table"], w.trees[i]["P"] = w.trees[i - 1]["table"], min(int(w.trees[i]["P"]), int(w.trees[i - 1]["P"]))
    _check(w, "diff_umma", tile_rows=64)


@gpu
def test_widening_follows_lengths_that_change_on_the_device():
    """A captured pass replayed after its trees and tiles were rewritten for longer sequences."""
    short, w = [(100, 20), (40, 4)], wl.make_pass("grown", 29, [(700, 20), (333, 4)], 8, 2, 128, 16, wl.BF16, wl.E4M3, scale=0.125)
    lam, norm_w = _weights(w, 3)
    op = host.AttnOp.for_workload(w, 32)
    dp = op.upload(w)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(op.device)
    trees = w.trees.copy()
    trees["P"] = [p for p, _ in short]
    plans = [host.plan_tiles(x, w.Hkv, mode=capi.ESP_PLAN_B200, split=0, tile_rows=32) for x in (trees, w.trees)]
    assert len(plans[0].tiles) == len(plans[1].tiles)
    O = torch.zeros((w.n_rows, w.q_ld), dtype=torch.int16, device=op.device)
    call = op.diff_call(plans[0], trees, dp.Q, dp.Kb, dp.Vb, O, kv=dp.kv, kv_scales=dp.kv_scales, blocks=dp.blocks, n_blocks=w.n_blocks, desc=dp.desc, lam=t(lam), norm_w=t(norm_w),
                        eps=EPS, out_scale=SCALE)
    op.diff_forward(call)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.diff_forward(call)
    tiles_dev, trees_dev = call.keep[2], call.keep[3]
    tiles_dev.copy_(t(plans[1].tiles.view(np.int32)).view_as(tiles_dev))
    trees_dev.copy_(t(w.trees.view(np.int32)).view_as(trees_dev))
    g.replay()
    torch.cuda.synchronize()
    op.check_status()
    O64, tol = diff64(w, lam, norm_w, EPS, SCALE, U16[wl.BF16])
    assert (np.abs(wl.from_bits16(O.cpu().numpy().view(np.uint16), wl.BF16).astype(np.float64) - O64) <= tol).all()
    op.close()


LAYOUTS = [  # trees (P, M), H, Hkv, options, tile_rows, split, kernel
    ("decode", [(100, 1), (0, 1), (333, 1)], 8, 2, None, 8, 32, "diff_decode"),
    ("rows", [(100, 20), (0, 140), (333, 7)], 8, 2, None, 128, 0, "diff_umma"),
    ("rows split", [(400, 20), (333, 7)], 8, 1, None, 16, 64, "diff_umma"),
    ("general", [(100, 3), (0, 9), (333, 1)], 8, 2, GENERAL, 8, 64, "diff_general"),
]


@gpu
@pytest.mark.parametrize("pool", [None, wl.E4M3], ids=["16-bit", "e4m3"])
@pytest.mark.parametrize("HD", [128, 256])
@pytest.mark.parametrize("case", LAYOUTS, ids=[c[0] for c in LAYOUTS])
def test_a_layer_inside_a_wider_pool(case, HD, pool):
    """The second of three layers of a pool whose rows, like the queries', the batch keys' and the output's, lie further apart than they are
    wide. Everything beside them is NaN, and stays as it was."""
    name, trees, H, Hkv, options, tile_rows, split, kernel = case
    w = wl.make_pass(name, 30, trees, H, Hkv, HD, 16, wl.BF16, pool, scale=(HD // 2) ** -0.5)
    q_ld, kv_ld, kv = w.q_ld + 72, w.kv_ld + 128, w.kv.reshape(-1, w.kv_ld)
    nan16, nan_pool = 0x7FC0, 0x7FC0 if pool is None else 0x7F

    def spread(x, ld, fill):
        out = np.full((x.shape[0], ld), fill, dtype=x.dtype)
        out[:, :x.shape[1]] = x
        return out

    lam, norm_w = _weights(w, 3)
    op = host.AttnOp.for_workload(w, tile_rows)
    for k, v in (options or {}).items():
        op.set_option(k, v)
    plan = host.plan_tiles(w.trees, Hkv, mode=capi.ESP_PLAN_B200, split=split, min_chunk=32, groups=4096 if split else 1, tile_rows=tile_rows)
    dp = op.upload(w)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a).view({2: np.int16, 1: np.uint8, 4: a.dtype}[a.dtype.itemsize])).to(op.device)
    call = op.diff_call(plan, w.trees, dp.Q, dp.Kb, dp.Vb, dp.O, kv=dp.kv, kv_scales=dp.kv_scales, blocks=dp.blocks, n_blocks=w.n_blocks, desc=dp.desc, lam=t(lam),
                        norm_w=t(norm_w), eps=EPS, out_scale=SCALE)
    layer = spread(kv, kv_ld, nan_pool)
    other = np.full_like(layer, nan_pool)
    wide = dict(Q=t(spread(w.Q, q_ld, nan16)), Kb=t(spread(w.Kb, kv_ld, nan16)), Vb=t(spread(w.Vb, kv_ld, nan16)), kv=t(np.concatenate([other, layer, other])),
                O=torch.full((w.n_rows, q_ld), 0x1234, dtype=torch.int16, device=op.device))
    scratch = torch.empty(len(w.blocks) * (2 * w.bt * kv_ld * 2 + 4) + 256, dtype=torch.uint8, device=op.device)
    for k, v in wide.items():
        setattr(call.args, k, v.data_ptr())
    call.args.p.q_ld, call.args.p.kv_ld, call.args.p.kv_base = q_ld, kv_ld, layer.size
    call.args.dequant_scratch, call.args.dequant_scratch_bytes = scratch.data_ptr(), scratch.numel()
    op.diff_forward(call)
    torch.cuda.synchronize()
    op.check_status()
    assert op.last_kernel == kernel
    O = wide["O"].cpu().numpy().view(np.uint16)
    op.close()
    assert (O[:, w.q_ld:] == 0x1234).all()
    O64, tol = diff64(w, lam, norm_w, EPS, SCALE, _unit(w, kernel))
    assert (np.abs(wl.from_bits16(O[:, :w.q_ld], wl.BF16).astype(np.float64) - O64) <= tol).all()


# ---------------------------------------------------------------------------------------------- without a GPU
def _append_args(**more):
    a = capi.AppendArgs(Q=0x10000, K=0x20000, V=0x30000, Qo=0x40000, Kb=0x50000, Vb=0x60000, kv=0x70000, kv_scales=0x80000, slots=0x90000, pos=0xA0000, inv_freq=0xB0000,
                        q_src_ld=1536, k_src_ld=1536, v_src_ld=1536, rows=4, maps=1, rot_half=64, n_blocks=9, qscale=1.0)
    a.p = capi.Params(8, 2, 1024, 256, 0, 16, 0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def _diff_args(trees, plan, /, **more):
    a = capi.Args(Q=0x10000, Kb=0x20000, Vb=0x30000, kv=0x40000, kv_scales=0x48000, blocks=0x50000, desc=0x60000, anc_mask=0x68000, O=0x70000, tiles=0x80000, trees=0x90000,
                  jobs=0x98000, tiles_host=plan.tiles.ctypes.data, trees_host=trees.ctypes.data, n_tiles=len(plan.tiles), n_trees=len(trees),
                  n_rows=int(trees["M"].sum()), n_blocks=9, n_block_entries=3)
    a.p = capi.Params(8, 2, 1024, 256, 2048, 16, 0)
    for k, v in more.items():
        setattr(a, k, v)
    return a


def test_misaligned_pointers_are_refused(call_checks):  # noqa: F811
    """What the kernels read in words of 4, 8 or 16 bytes has to lie on their multiples: anything else faults on the device."""
    shape = capi.Shape(8, 2, 128, 16, wl.BF16, wl.E4M3, 8, 0, 0.125)
    assert call_checks.append(shape, _append_args()) == 0
    for name in ("pos", "inv_freq", "kv_scales"):
        for off in (1, 2):
            assert call_checks.append(shape, _append_args(**{name: getattr(_append_args(), name) + off})) == capi.ESP_ERR_INVALID, name
    trees = host.make_trees([4, 1], [20, 3], [0, 2])
    plan = host.plan_tiles(trees, 2)
    good, d = _diff_args(trees, plan), capi.DiffArgs(0x100000, 0x110000, 0, 1e-5, 1.0)
    assert call_checks.diff(shape, good, d) == 0
    for name, unit in (("tiles", 16), ("trees", 16), ("desc", 16), ("anc_mask", 8), ("jobs", 4), ("blocks", 4), ("kv_scales", 4)):
        assert call_checks.diff(shape, _diff_args(trees, plan, **{name: getattr(good, name) + unit // 2}), d) == capi.ESP_ERR_INVALID, name
        assert call_checks.diff(shape, _diff_args(trees, plan, **{name: getattr(good, name) + unit}), d) == 0, name
    assert call_checks.diff(shape, good, capi.DiffArgs(0x100002, 0x110000, 0, 1e-5, 1.0)) == capi.ESP_ERR_INVALID


def _bare(kv_dtype=wl.BF16):
    """An AttnOp without a context: it makes calls of CPU tensors, which nothing here launches."""
    op = object.__new__(host.AttnOp)
    op.lib, op.device, op.shape = capi.load(), torch.device("cpu"), capi.Shape(8, 2, 128, 16, wl.BF16, kv_dtype, 8, 0, 0.125)
    return op




@pytest.mark.parametrize("pool", [wl.BF16, wl.E4M3], ids=["16-bit", "e4m3"])
def test_append_tensors_of_other_types_and_lengths_are_refused(pool):
    """The kernel reads rows of its own types from the addresses it gets: another type is read as garbage, a shorter tensor past its end."""
    op, n, z = _bare(pool), 5, torch.zeros
    kv = z(9 * 2 * 16 * 256, dtype=torch.uint8 if pool == wl.E4M3 else torch.bfloat16)
    good = dict(Q=z(n, 1024, dtype=torch.bfloat16), K=z(n, 256, dtype=torch.bfloat16), V=z(n, 256, dtype=torch.bfloat16), Qo=z(n, 1024, dtype=torch.bfloat16),
                Kb=z(n, 256, dtype=torch.bfloat16), Vb=z(n, 256, dtype=torch.bfloat16), kv=kv, kv_scales=z(9, 2, 2) if pool == wl.E4M3 else None, n_blocks=9,
                slots=z(n, 2, dtype=torch.int32), pos=z(n, dtype=torch.int32), inv_freq=z(64))
    more = [(name, good[name].to(t)) for name in ("Q", "V", "Qo", "Kb", "Vb") for t in (torch.float16, torch.float32, torch.int32)]
    more += [(name, good[name][:n - 1]) for name in ("Q", "V", "Qo", "Kb", "Vb", "slots", "pos")]
    more += [(name, good[name][:, :255]) for name in ("Q", "K", "V", "Qo")] + [("Kb", good["Kb"][:, :128]), ("Vb", good["Vb"][:, :128].contiguous())]
    more += [("slots", good["slots"].long()), ("pos", good["pos"].long()), ("pos", z(2 * n, dtype=torch.int32)[::2]), ("inv_freq", good["inv_freq"].double()),
             ("inv_freq", z(128)[::2]), ("kv", kv[1:]), ("kv", kv.float()), ("n_blocks", 10)]
    if pool == wl.E4M3:
        more += [("kv_scales", z(8, 2, 2)), ("kv_scales", z(9, 2, 2).double())]
    more += [(name, torch.empty_like(good[name], device="meta")) for name in ("Q", "K", "V", "Qo", "Kb", "Vb", "kv", "slots", "pos", "inv_freq")]
    for name, bad in more:
        call = dict(good, **{name: bad})
        with pytest.raises(ValueError, match="^(kv|K|V|Q|%s)" % name):  # a wrong K may show at the tensors that have to go with it
            op.append_call(**call)
    op.append_call(**good)
    f32 = {k: good[k].float() for k in "QKV"}
    assert op.append_call(**dict(good, **f32)).args.src_f32 == 1
    bits = {k: good[k].view(torch.int16) for k in ("Q", "K", "V", "Qo", "Kb", "Vb")}
    assert op.append_call(**dict(good, **bits)).args.src_f32 == 0
    assert op.append_call(None, good["K"], good["V"], Kb=good["Kb"], Vb=good["Vb"]).args.rot_half == 0


@pytest.mark.parametrize("pool", [wl.BF16, wl.E4M3], ids=["16-bit", "e4m3"])
def test_attention_tensors_of_other_types_and_lengths_are_refused(pool):
    op, n, z = _bare(pool), 5, torch.zeros
    trees = host.make_trees([4, 1], [200, 3], [0, 13])
    plan = host.plan_tiles(trees, 2, mode=capi.ESP_PLAN_B200, split=1 << 20, min_chunk=16, groups=64)
    assert plan.n_parts
    kv = z(9 * 2 * 16 * 256, dtype=torch.uint8 if pool == wl.E4M3 else torch.int16)
    parts = int(op.lib.esp_diff_parts_floats(C.byref(op.shape), plan.n_parts))
    good = dict(Q=z(n, 1024, dtype=torch.bfloat16), Kb=z(n, 256, dtype=torch.bfloat16), Vb=z(n, 256, dtype=torch.int16), O=z(n, 1024, dtype=torch.bfloat16), kv=kv, n_blocks=9,
                kv_scales=z(9, 2, 2) if pool == wl.E4M3 else None, blocks=z(14, dtype=torch.int32), desc=z(n, 4, dtype=torch.int32), anc_mask=z(n, dtype=torch.int64), lam=z(8),
                norm_w=z(128), parts=z(parts), scratch=z(8, dtype=torch.uint8))
    more = [(name, good[name].to(t)) for name in ("Q", "Kb", "Vb", "O") for t in (torch.float16, torch.float32, torch.int64)]
    more += [(name, good[name][:n - 1]) for name in ("Kb", "Vb", "O", "desc", "anc_mask")] + [("O", good["O"][:, :1016]), ("Q", z(n, 1016, dtype=torch.bfloat16))]
    more += [("blocks", good["blocks"].long()), ("desc", good["desc"].long()), ("desc", good["desc"].t()), ("anc_mask", good["anc_mask"].int()), ("lam", z(7)), ("lam", z(8).double()),
             ("norm_w", z(127)), ("norm_w", z(128, dtype=torch.bfloat16)), ("parts", z(parts - 1)), ("parts", z(parts).double()), ("kv", kv[1:]), ("kv", kv.float()),
             ("scratch", z(8)), ("kv_scales", z(8, 2, 2)), ("kv_scales", z(9, 2, 2).half())]
    more += [(name, torch.empty_like(t, device="meta")) for name, t in good.items() if isinstance(t, torch.Tensor)]
    for name, bad in more:
        with pytest.raises(ValueError, match="^(O|%s)" % name):
            op.diff_call(plan, trees, **dict(good, **{name: bad}))
    op.diff_call(plan, trees, **good)
    op.diff_call(plan, trees, **dict(good, lam=z(n, 8), lam_ld=8))
    with pytest.raises(ValueError, match="^lam"):
        op.diff_call(plan, trees, **dict(good, lam=z(n - 1, 8), lam_ld=8))


def test_lambda_vectors_laid_out_differently_are_refused():
    op, z = _bare(), torch.zeros
    for more in (dict(k1=z(8, 65)[:, :64]), dict(q2=z(7, 64)), dict(k2=z(8, 64).half()), dict(q1=z(64)), dict(k1=z(64, 8).t())):
        v = dict(dict(q1=z(8, 64), k1=z(8, 64), q2=z(8, 64), k2=z(8, 64)), **more)
        with pytest.raises(ValueError, match="^[qk][12]"):
            op.diff_lambda(lambda_init=0.1, **v)
    with pytest.raises(ValueError, match="^q1"):
        op.diff_lambda(z(4, 64), z(4, 64), z(4, 64), z(4, 64), lambda_init=0.1)


def _planned(rows, cached, H, Hkv, HD, kv_dtype=wl.BF16):
    """(tile rows, parts of the longest list) that the options give."""
    trees = host.make_trees(rows, cached, [0] * len(rows))
    tile_rows, opts = host.diff_plan_options(trees, H, Hkv, HD, kv_dtype)
    plan = host.plan_tiles(trees, Hkv, **opts)
    return tile_rows, int(max(plan.jobs["nparts"])) if len(plan.jobs) else 1


def test_few_rows_behind_a_long_prefix_share_tiles_and_split():
    """One user's draft tree: the heads of a kv head share a tile, and the prefix is cut for the whole GPU."""
    for rows, cached, HD in ((16, 16384, 128), (5, 32768, 128), (16, 16384, 256)):
        tile_rows, parts = _planned([rows], [cached], 32, 4, HD)
        assert tile_rows == 16 and parts >= 16, (rows, cached, HD, tile_rows, parts)
    # what was planned well before stays: prompts in tiles of one head, a chunk in two parts, a batch of trees unsplit
    assert _planned([8192] * 2, [0] * 2, 16, 4, 128) == (128, 1)
    assert _planned([700], [20001], 32, 8, 128, wl.E4M3) == (64, 2)
    assert _planned([16] * 16, [4096] * 16, 32, 4, 128) == (16, 1)


def test_single_rows_of_many_heads_are_planned_for_tiles_that_run_fast():
    """diff_decode takes 8 heads to a kv head; tiles of 8 rows would leave the rest to diff_general."""
    for H, Hkv, rows in ((32, 2, 16), (32, 1, 16), (12, 1, 32), (9, 1, 128)):
        for kv_dtype in (wl.BF16, wl.E4M3):
            assert _planned([1] * 8, [4096] * 8, H, Hkv, 128, kv_dtype)[0] == rows, (H, Hkv)
    assert _planned([1], [4096], 32, 4, 128)[0] == 8 and _planned([1], [4096], 32, 1, 64)[0] == 8


def test_idle_slots_do_not_change_the_plan():
    for rows, cached in (([1] * 31, [4096] * 31), ([1], [100]), ([16] * 3, [4096, 9000, 5]), ([300], [0])):
        idle_rows, idle_cached = [0] + rows + [0, 0], [700] + cached + [0, 4096]
        assert _planned(idle_rows, idle_cached, 32, 4, 128) == _planned(rows, cached, 32, 4, 128)


def test_plan_options_of_the_largest_passes():
    """Counts near 2^31 do not wrap: 2^24 tiles and more want as many places."""
    for cached, H in ((0, 128), (2 ** 31 - 1, 256)):
        tile_rows, o = host.diff_plan_options(host.make_trees([2 ** 31 - 1], [cached], [0]), H, 128, 128, wl.BF16)
        assert tile_rows == 128 and o["groups"] >= 2 ** 24


def test_plans_know_the_type_of_the_pool():
    """A context plans for its own pool: 131072 E4M3 keys of 8 kv heads and 256 dims for two CTAs to an SM, 16-bit ones for one. Passes that want
    another tile height are refused."""
    step, prompt = host.make_trees([1], [131072], [0]), host.make_trees([700], [0], [0])
    for kv_dtype, ctas in ((wl.E4M3, 296), (wl.BF16, 148)):
        op = _bare(kv_dtype)
        op.shape = capi.Shape(32, 8, 256, 16, wl.BF16, kv_dtype, 8, 0, 0.088)
        plan = op.diff_plan(step)
        assert ctas - 8 <= len(plan.tiles) * 8 <= ctas and plan.tile_rows == 8
        with pytest.raises(ValueError, match="tile_rows=128, not 8"):
            op.diff_plan(prompt)
        op.shape.tile_rows = 128
        assert op.diff_plan(prompt).tile_rows == 128
