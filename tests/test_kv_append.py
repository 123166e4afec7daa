"""esp_kv_append against its 64-bit form: types, head layouts, both pairings, odd rotary widths, strides, padding rows, far
positions, writing over its sources, both pool types; refusals; and slots outside the pool."""
import numpy as np
import pytest
import torch

from espetero_b200 import capi, host, workloads as wl

from .diff_ref import SUB16, U16, call_checks, rotate64  # noqa: F401 (a fixture)

T16 = {wl.F16: torch.float16, wl.BF16: torch.bfloat16}
gpu = pytest.mark.gpu


def _bits(t):
    return t.cpu().view(torch.int16).numpy().view(np.uint16)


def _case(rows, H, Hkv, HD, maps, rot_half, adjacent, q_dtype, src32, pool, seed, bt=16, pad=0, lead=0, far=False):
    rng = np.random.default_rng(seed)
    wide = (H + 2 * Hkv) * HD + lead
    X = rng.standard_normal((rows, wide)).astype(np.float32)
    if not src32:
        X = wl.from_bits16(wl.to_bits16(X, q_dtype), q_dtype)
    n_blocks = (rows + bt - 1) // bt + 2
    order = rng.permutation(n_blocks)
    slots = np.stack([order[np.arange(rows) // bt], np.arange(rows) % bt], axis=1).astype(np.int32)
    slots[rng.permutation(rows)[:pad], 0] = -1
    pos = (np.arange(rows) + (2 ** 30 if far else 131000)).astype(np.int32)
    inv = (10000.0 ** (-np.arange(rot_half) / max(rot_half, 1))).astype(np.float32)
    scales = np.exp2(rng.uniform(-7, 0, size=(n_blocks, 2, Hkv))).astype(np.float32) if pool == wl.E4M3 else None
    return dict(rows=rows, H=H, Hkv=Hkv, HD=HD, maps=maps, adjacent=adjacent, q_dtype=q_dtype, src32=src32, pool=pool, bt=bt, lead=lead, X=X,
                n_blocks=n_blocks, slots=slots, pos=pos, inv=inv, scales=scales, kv_base=2 * 5 * bt * Hkv * HD)


def _run(c, with_q=True, with_batch=True, in_place=False, stream=None, qscale=0.25):
    dev = torch.device("cuda", 0)
    op = host.AttnOp(c["H"], c["Hkv"], c["HD"], c["bt"], c["q_dtype"], c["pool"], 1.0)
    t = lambda a: None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev)
    X = t(c["X"])
    X = X if c["src32"] else X.to(T16[c["q_dtype"]])
    q, k, v = X[:, c["lead"]:].split([c["H"] * c["HD"], c["Hkv"] * c["HD"], c["Hkv"] * c["HD"]], dim=1)
    if in_place:
        q, k, v = (x.contiguous() for x in (q, k, v))
    kv_ld, dt = c["Hkv"] * c["HD"], T16[c["q_dtype"]]
    Qo = q if in_place else torch.zeros((c["rows"], c["H"] * c["HD"]), dtype=dt, device=dev)
    Kb, Vb = (k, v) if in_place else (torch.zeros((c["rows"], kv_ld), dtype=dt, device=dev) for _ in range(2))
    n = c["kv_base"] + c["n_blocks"] * 2 * c["bt"] * kv_ld
    pool = torch.full((n,), 0x31, dtype=torch.uint8, device=dev) if c["pool"] == wl.E4M3 else torch.full((n,), 0x3131, dtype=torch.int16, device=dev)
    call = op.append_call(q if with_q else None, k, v, Qo if with_q else None, Kb if with_batch else None, Vb if with_batch else None, kv=pool, kv_scales=t(c["scales"]),
                          n_blocks=c["n_blocks"], slots=t(c["slots"]), pos=t(c["pos"]), inv_freq=t(c["inv"]) if len(c["inv"]) else None, maps=c["maps"],
                          adjacent=c["adjacent"], qscale=qscale, kv_base=c["kv_base"])
    torch.cuda.synchronize()
    op.kv_append(call, stream)
    torch.cuda.synchronize()
    op.check_status()
    out = _bits(Qo), _bits(Kb), _bits(Vb), pool.cpu().numpy()
    op.close()
    return out


def _check(c, got, with_q=True, with_batch=True, qscale=0.25):
    Qo, Kb, Vb, pool = got
    H, Hkv, HD, rows = c["H"], c["Hkv"], c["HD"], c["rows"]
    X = c["X"][:, c["lead"]:].astype(np.float64)
    u = U16[c["q_dtype"]]
    refs = []
    for x, heads, f in ((X[:, :H * HD], H, qscale), (X[:, H * HD:(H + Hkv) * HD], Hkv, 1.0)):
        y, mag = rotate64(x.reshape(rows, heads, HD), c["pos"], c["inv"], c["maps"], c["adjacent"])
        # two products and a sum (3 * 2^-24), cosine and sine good to 4 * 2^-24, the angle's fraction of a turn held in fp32
        # (pi 2^-24), one product with qscale: under 16 * 2^-24 of |x| + |y|; then one rounding to 16 bits
        refs.append((f * y, u * np.abs(f * y) * (1 + 2.0 ** -9) + (1 + u) * 16 * 2.0 ** -24 * np.abs(f) * mag + SUB16[c["q_dtype"]]))
    if with_q:
        err = np.abs(wl.from_bits16(Qo, c["q_dtype"]).reshape(rows, H, HD).astype(np.float64) - refs[0][0])
        assert (err <= refs[0][1]).all(), float((err - refs[0][1]).max())
    if with_batch:
        err = np.abs(wl.from_bits16(Kb, c["q_dtype"]).reshape(rows, Hkv, HD).astype(np.float64) - refs[1][0])
        assert (err <= refs[1][1]).all(), float((err - refs[1][1]).max())
        assert np.array_equal(Vb, wl.to_bits16(c["X"][:, c["lead"] + (H + Hkv) * HD:], c["q_dtype"]))
        # the pool: exactly the rounded rows (or their codes) at their slots, and nothing else
        expect = np.full_like(pool, 0x31 if c["pool"] == wl.E4M3 else 0x3131)
        body = expect[c["kv_base"]:].reshape(c["n_blocks"], 2, c["bt"], Hkv, HD)
        for r in range(rows):
            b, s = c["slots"][r]
            if b < 0:
                continue
            for which, x in ((0, Kb), (1, Vb)):
                row = x[r].reshape(Hkv, HD)
                body[b, which, s] = (wl.e4m3_encode((wl.from_bits16(row, c["q_dtype"]) / c["scales"][b, which][:, None]).astype(np.float32))
                                     if c["pool"] == wl.E4M3 else row.view(np.int16))
        assert np.array_equal(pool, expect)


# rows, H, Hkv, HD, maps, rot_half, adjacent, type, fp32 source, pool, more
CASES = [
    (1, 8, 2, 128, 2, 32, False, wl.BF16, False, wl.BF16, {}),
    (1, 8, 2, 128, 1, 64, True, wl.F16, False, wl.F16, {}),
    (37, 4, 4, 64, 1, 32, False, wl.F16, True, wl.F16, {}),
    (37, 4, 2, 64, 2, 16, True, wl.BF16, False, wl.E4M3, dict(pad=5)),
    (300, 32, 8, 256, 2, 64, False, wl.BF16, False, wl.E4M3, dict(pad=11)),
    (129, 6, 2, 256, 1, 32, False, wl.BF16, True, wl.BF16, dict(bt=24)),
    (5, 2, 1, 512, 1, 256, True, wl.F16, False, wl.F16, {}),
    (9, 2, 1, 512, 2, 128, False, wl.BF16, False, wl.E4M3, {}),
    (19, 4, 2, 128, 1, 48, False, wl.BF16, False, wl.BF16, {}),       # not a power of two, passes some dims through
    (19, 4, 2, 128, 2, 13, False, wl.BF16, False, wl.E4M3, {}),       # odd width: one-dim items
    (19, 4, 2, 128, 1, 13, True, wl.F16, True, wl.E4M3, {}),          # odd width, adjacent
    (19, 4, 2, 128, 1, 13, True, wl.BF16, False, wl.BF16, {}),
    (23, 4, 2, 128, 2, 32, False, wl.F16, False, wl.F16, dict(lead=3)),  # rows that start at no 16-byte boundary
    (23, 4, 2, 128, 2, 32, True, wl.BF16, True, wl.BF16, dict(lead=5)),
    (11, 4, 2, 128, 1, 0, False, wl.BF16, False, wl.BF16, {}),        # no rotation
    (64, 4, 2, 128, 1, 64, False, wl.F16, False, wl.F16, dict(far=True)),
    (3000, 1, 1, 64, 1, 32, False, wl.F16, False, wl.F16, {}),        # many rows per CTA
]


@gpu
@pytest.mark.parametrize("i", range(len(CASES)))
def test_append_matches_64_bits(i):
    c = _case(*CASES[i][:10], seed=i, **CASES[i][10])
    _check(c, _run(c))


@gpu
def test_append_over_its_sources():
    c = _case(50, 8, 2, 128, 2, 32, False, wl.BF16, False, wl.BF16, seed=90)
    _check(c, _run(c, in_place=True))
    c = _case(50, 8, 2, 128, 2, 13, True, wl.F16, False, wl.E4M3, seed=91)
    _check(c, _run(c, in_place=True))


@gpu
def test_append_keys_and_values_alone():
    c = _case(33, 8, 2, 128, 1, 64, False, wl.BF16, False, wl.E4M3, seed=92)
    full, kv_only, pool_only = _run(c), _run(c, with_q=False), _run(c, with_q=False, with_batch=False)
    _check(c, kv_only, with_q=False)
    assert np.array_equal(full[3], kv_only[3]) and np.array_equal(full[3], pool_only[3])
    assert not kv_only[0].any() and not pool_only[1].any()


@gpu
def test_append_gives_the_codes_of_kv_save():
    """Append with a pool, and append without one followed by esp_kv_save, leave the same bytes."""
    c = _case(40, 8, 4, 128, 1, 64, False, wl.BF16, False, wl.E4M3, seed=93)
    _, Kb, Vb, pool = _run(c)
    w = wl.make_pass("save", 1, [(0, 40)], 8, 4, 128, 16, wl.BF16, wl.E4M3)
    w.Kb, w.Vb, w.kv_base = Kb, Vb, c["kv_base"]
    w.kv, w.kv_scales, w.n_blocks = np.full(pool.size, 0x31, dtype=np.uint8), c["scales"], c["n_blocks"]
    op = host.AttnOp.for_workload(w)
    dp = op.upload(w)
    entries = np.zeros(40, dtype=wl.KVSAVE_DT)
    entries["src_row"], entries["block"], entries["pos"] = np.arange(40), c["slots"][:, 0], c["slots"][:, 1]
    keep = op.kv_save(dp, entries)
    torch.cuda.synchronize()
    assert np.array_equal(dp.kv.cpu().numpy(), pool)
    op.close()


@gpu
def test_append_beside_the_current_stream_and_in_a_graph():
    c = _case(65, 8, 2, 128, 2, 32, False, wl.BF16, False, wl.BF16, seed=94)
    want = _run(c)
    side = torch.cuda.Stream()
    got = _run(c, stream=side.cuda_stream)
    assert all(np.array_equal(a, b) for a, b in zip(want, got))
    # captured once, replayed on new inputs in the same buffers
    dev = torch.device("cuda", 0)
    op = host.AttnOp(8, 2, 128, 16, wl.BF16, wl.BF16, 1.0)
    X = torch.zeros((65, 12 * 128), dtype=torch.bfloat16, device=dev)
    q, k, v = X.split([1024, 256, 256], dim=1)
    Qo = torch.zeros((65, 1024), dtype=torch.bfloat16, device=dev)
    Kb, Vb = torch.zeros((65, 256), dtype=torch.bfloat16, device=dev), torch.zeros((65, 256), dtype=torch.bfloat16, device=dev)
    pool = torch.full((c["kv_base"] + c["n_blocks"] * 2 * 16 * 256,), 0x3131, dtype=torch.int16, device=dev)
    t = lambda a: torch.from_numpy(a).to(dev)
    call = op.append_call(q, k, v, Qo, Kb, Vb, kv=pool, n_blocks=c["n_blocks"], slots=t(c["slots"]), pos=t(c["pos"]), inv_freq=t(c["inv"]), maps=2, qscale=0.25,
                          kv_base=c["kv_base"])
    op.kv_append(call)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        op.kv_append(call)
    X.copy_(t(c["X"]).to(torch.bfloat16))
    g.replay()
    torch.cuda.synchronize()
    assert all(np.array_equal(a, b) for a, b in zip(want, (_bits(Qo), _bits(Kb), _bits(Vb), pool.cpu().numpy())))
    op.close()


@gpu
def test_append_reports_a_slot_outside_the_pool():
    """A block id past the region and a position past the page: not written, and the status word says so."""
    c = _case(20, 8, 2, 128, 1, 64, False, wl.BF16, False, wl.BF16, seed=95)
    good = _run(c)
    for bad in ((c["n_blocks"], 0), (0, 16), (0, -1)):
        d = dict(c, slots=c["slots"].copy())
        d["slots"][7] = bad
        with pytest.raises(capi.EspError, match="bad block id"):
            _run(d)
    d = dict(c, slots=c["slots"].copy())
    d["slots"][7, 0] = -1  # the same row as padding: everything else as before
    got = _run(d)
    assert all(np.array_equal(a, b) for a, b in zip(good[:3], got[:3]))
    assert (good[3] != got[3]).sum() <= 2 * 256


# ---------------------------------------------------------------------------------------------- refusals (no GPU needed)
SHAPE = dict(H=8, Hkv=2, HD=128, bt=16, q_dtype=wl.BF16, kv_dtype=wl.BF16)
GOOD = dict(Q=0x10000, K=0x20000, V=0x30000, Qo=0x40000, Kb=0x50000, Vb=0x60000, kv=0x70000, kv_scales=0x80000, slots=0x90000, pos=0xA0000, inv_freq=0xB0000,
            q_src_ld=1536, k_src_ld=1536, v_src_ld=1536, rows=4, src_f32=0, maps=1, rot_half=64, adjacent=0, n_blocks=9, qscale=1.0)
REFUSED = [dict(K=0), dict(V=0), dict(Qo=0), dict(kv=0, Kb=0), dict(maps=0), dict(maps=3), dict(rot_half=65), dict(rot_half=-1), dict(maps=2, rot_half=33),
           dict(pos=0), dict(inv_freq=0), dict(q_src_ld=1023), dict(k_src_ld=255), dict(K=0x20001), dict(src_f32=1, V=0x30002), dict(slots=0), dict(slots=0x90004),
           dict(n_blocks=0), dict(kv=0x70008), dict(Kb=0x50001), dict(rows=-1), dict(src_f32=2), dict(Qo=0x10000), dict(Vb=0x30000, src_f32=1)]


def test_append_refuses_bad_arguments(call_checks):
    shape = capi.Shape(**{k: SHAPE[k] for k in ("H", "Hkv", "HD", "bt", "q_dtype", "kv_dtype")}, tile_rows=8, flags=0, scale=1.0)

    def code(**more):
        a = capi.AppendArgs(**{**GOOD, **more})
        a.p = capi.Params(8, 2, 1024, 256, 0, 16, 0)
        return call_checks.append(shape, a)

    assert code() == 0
    assert code(rows=0, K=0) == 0
    assert code(rot_half=0, pos=0, inv_freq=0) == 0
    assert code(Q=0, Qo=0) == 0
    assert code(kv=0) == 0 and code(Kb=0, Vb=0) == 0
    for more in REFUSED:
        assert code(**more) == capi.ESP_ERR_INVALID, more
    shape.kv_dtype = wl.E4M3
    assert code() == 0 and code(kv_scales=0) == capi.ESP_ERR_INVALID


def test_append_needs_a_context():
    lib = capi.load()
    assert lib.esp_kv_append(None, None, capi.AppendArgs()) == capi.ESP_ERR_INVALID
