"""GPU parity of the operators around a draft tree, through the C ABI: normed and rotated append, tree attention, log
probabilities, row copies, each against a plain implementation in 64 bits with tolerances counted from the roundings
(plain_operators.py), and the loop of all of them, eager and as a replayed graph."""
import numpy as np
import pytest

import backburner_amd as bb
import oracle as orc
import plain_operators as plain

pytestmark = pytest.mark.gpu
F16, Q8, Q4 = bb.FMT_F16, bb.FMT_Q8_0, bb.FMT_Q4_0


@pytest.fixture(scope="module")
def ws():
    w = bb.Workspace()
    yield w
    w.close()


def buf(a):
    return bb.DeviceBuffer.from_array(np.ascontiguousarray(a))


# ---------------------------------------------------------------- tree attention
def run_tree(ws, shape, K, V, counts, Q, n_nodes, mask, stream=None):
    """(Oh, lse) of the call over pages of `counts` keys; outputs start poisoned."""
    pg = bb.pages_from_rows(K, V, shape.rs, list(counts))
    rows = shape.nkv * shape.rows
    dq, dm = buf(Q.astype(np.float32)), buf(mask.astype(np.uint64))
    do, dl = buf(np.full(rows * shape.hd + 64, 0x7e11, np.uint16)), buf(np.full(rows + 16, 7.0, np.float32))
    try:
        ws.attn_tree(shape, pg, n_nodes, dm.ptr, dq.ptr, do.ptr, dl.ptr, stream)
        if stream:
            assert bb.synth().pa_synth_stream_sync(stream) == 0
        bb.device_sync()
        o, l = do.download(np.uint16), dl.download(np.float32)
        assert np.all(o[rows * shape.hd:] == 0x7e11) and np.all(l[rows:] == 7.0)   # nothing behind the last row
        return o[:rows * shape.hd].reshape(rows, shape.hd), l[:rows]
    finally:
        for b in (dq, dm, do, dl):
            b.close()
        pg.close()


def check_tree(shape, K, V, n, Q, n_nodes, mask, got):
    o, lse, tol_o, tol_l = plain.attn_tree(shape, K, V, n, Q, n_nodes, mask)
    oh = got[0].view(np.float16).astype(np.float64)
    dead = np.isneginf(lse)
    assert np.all(oh[dead] == 0) and np.all(np.isneginf(got[1][dead]))
    live = ~dead
    assert np.all(np.isfinite(oh[live])) and np.all(np.isfinite(got[1][live]))
    eo, el = np.abs(oh - o)[live] / tol_o[live], np.abs(got[1][live] - lse[live]) / tol_l[live]
    if live.any():
        print(f"  of the tolerance: O {eo.max():.2f} lse {el.max():.2f}", flush=True)
        assert eo.max() <= 1 and el.max() <= 1


def tree_case(seed, fmt, nkv, gqa, hd, nodes, n, pad=0):
    rng = np.random.default_rng(seed)
    hb = orc.head_bytes(fmt, hd); rs = nkv * hb + pad
    K = orc.fill_rows(seed, fmt, nkv, hd, n, rs=rs, n_outliers=4, outlier_mul=8.0)
    V = orc.fill_rows(seed + 1, fmt, nkv, hd, n, rs=rs)
    Q = orc.normal(seed + 2, 0, nkv * gqa * nodes * hd).reshape(nkv * gqa * nodes, hd)
    return rng, bb.make_shape(nkv, gqa * nodes, hd, fmt, rs=rs), K, V, Q


def split_pages(rng, n, page):
    if page == "one":
        return [n]
    if page == "ragged":                                              # sizes from 0 up, the tree over many of them
        out, left = [], n
        while left:
            out.append(min(left, int(rng.integers(0, 41))))
            left -= out[-1]
        return out + [0]
    return [min(page, n - i) for i in range(0, n, page)]


# rows of a head from 1 to 512: the decode kernel, one and two tile streams, 4- and 8-wave kernels, several row blocks
TREES = [
    # fmt, nkv, gqa, hd, nodes, context, pages
    (Q8, 8, 8, 128, 1, 4096, 4096), (Q4, 8, 8, 128, 1, 500, 200), (F16, 8, 8, 128, 1, 300, "one"),
    (Q8, 2, 4, 128, 2, 33, "one"), (Q4, 2, 1, 128, 5, 1000, "ragged"), (F16, 2, 1, 128, 7, 31, "ragged"),
    (Q8, 8, 8, 128, 26, 2000, 1000), (Q4, 8, 8, 128, 26, 2007, 1000), (F16, 8, 8, 128, 26, 1990, 1000),
    (Q8, 1, 7, 128, 33, 1, "ragged"), (Q4, 3, 7, 128, 33, 100, "ragged"), (F16, 3, 5, 128, 17, 64, "ragged"),
    (Q8, 2, 8, 128, 64, 900, "one"), (Q4, 2, 8, 128, 64, 900, 64), (F16, 2, 8, 128, 64, 900, "ragged"),
    (Q8, 2, 6, 256, 1, 700, "one"), (Q8, 2, 6, 256, 8, 700, 256), (Q4, 2, 6, 256, 8, 701, 256), (F16, 2, 6, 256, 8, 702, 256),
    (Q8, 1, 8, 256, 64, 300, "ragged"), (Q4, 1, 8, 256, 64, 300, "ragged"), (F16, 1, 8, 256, 64, 300, "ragged"),
    # no context at all, one key of it, and a tree longer than every page
    (Q8, 2, 8, 128, 12, 0, "one"), (Q4, 2, 6, 256, 12, 0, "ragged"), (F16, 2, 8, 128, 64, 0, 5), (Q8, 8, 8, 128, 1, 0, "one"),
    (Q4, 2, 4, 128, 3, 1, 1), (Q8, 2, 2, 128, 64, 40, 1),
]


@pytest.mark.parametrize("fmt,nkv,gqa,hd,nodes,context,page", TREES)
def test_tree(ws, fmt, nkv, gqa, hd, nodes, context, page):
    n = context + nodes
    seed = 1000 + hd + 7 * nodes + context + fmt
    print(f"tree fmt={fmt} nkv={nkv} gqa={gqa} hd={hd} nodes={nodes} context={context} page={page}", flush=True)
    rng, shape, K, V, Q = tree_case(seed, fmt, nkv, gqa, hd, nodes, n)
    _, mask = plain.random_tree(rng, nodes)
    check_tree(shape, K, V, n, Q, nodes, mask, run_tree(ws, shape, K, V, split_pages(rng, n, page), Q, nodes, mask))


@pytest.mark.parametrize("fmt", [Q8, Q4, F16])
@pytest.mark.parametrize("hd,context", [(128, 0), (128, 77), (256, 0), (256, 77)])
def test_tree_masks(ws, fmt, hd, context):
    """Any mask, not trees alone: nothing, everything, one other node, random bits, a chain; bits past the nodes count for nothing. A
    row without context whose mask is empty sees no key."""
    nodes, nkv, gqa = 40, 2, 3
    print(f"tree masks fmt={fmt} hd={hd} context={context}", flush=True)
    rng, shape, K, V, Q = tree_case(50 + fmt + hd + context, fmt, nkv, gqa, hd, nodes, context + nodes)
    mask = rng.integers(0, 1 << 40, nodes, dtype=np.uint64)
    mask[0], mask[1], mask[2], mask[3] = 0, (1 << 40) - 1, 1 << 39, (1 << 64) - (1 << 40)
    mask[10:20] = [(1 << (i + 1)) - 1 for i in range(10, 20)]
    mask[20:30] |= np.uint64(0xabcdef << 40)
    got = run_tree(ws, shape, K, V, [context + nodes], Q, nodes, mask)
    check_tree(shape, K, V, context + nodes, Q, nodes, mask, got)
    dead = np.isneginf(got[1]).sum()
    assert dead == (2 * nkv * gqa if context == 0 else 0)


@pytest.mark.parametrize("what", ["nan", "inf", "-inf"])
@pytest.mark.parametrize("fmt", [Q8, Q4, F16])
def test_tree_unseen_bytes_do_not_count(ws, fmt, what):
    """Infinities and NaN in the key and value rows of nodes that some rows do not see: those rows keep their results bit for
    bit; rows that see a NaN value give NaN."""
    nodes, nkv, gqa, hd, context = 24, 2, 8, 128, 50
    print(f"tree unseen fmt={fmt} {what}", flush=True)
    rng, shape, K, V, Q = tree_case(70 + fmt, fmt, nkv, gqa, hd, nodes, context + nodes)
    _, mask = plain.random_tree(rng, nodes)
    mask[9] = 0
    bad = [5, 9, 23]
    want = run_tree(ws, shape, K, V, [60, 14], Q, nodes, mask)
    bits = {"nan": 0x7e00, "inf": 0x7c00, "-inf": 0xfc00}[what]
    for X in (K, V):
        for j in bad:
            row = X[(context + j) * shape.rs:(context + j + 1) * shape.rs]
            if fmt == F16:
                row.view(np.uint16)[:] = bits
            else:                                                     # every block scale
                b = row.reshape(-1, 34 if fmt == Q8 else 18)
                b[:, 0], b[:, 1] = bits & 0xff, bits >> 8
    got = run_tree(ws, shape, K, V, [60, 14], Q, nodes, mask)
    clean = np.array([not any(int(mask[r % nodes]) >> j & 1 for j in bad) for r in range(shape.nkv * shape.rows)])
    assert clean.any() and not clean.all()
    assert np.array_equal(got[0][clean], want[0][clean]) and np.array_equal(got[1][clean], want[1][clean])
    if what == "nan":
        assert np.all(np.isnan(got[0].view(np.float16)[~clean]))


@pytest.mark.parametrize("fmt,nkv,gqa,nodes,context,page", [
    (Q8, 1, 8, 8, 90000, 4096),                                       # 64 rows, long chunks: two tile streams
    (Q4, 1, 8, 5, 150000, 4096),                                      # 40 rows
    (F16, 1, 4, 8, 90000, 4096),                                      # 32 rows
    (Q8, 2, 4, 2, 40000, 200),                                        # 201 pages: the decode kernel in two launches
    (Q4, 2, 8, 4, 9000, 64),                                          # 141 pages
])
def test_tree_long_context(ws, fmt, nkv, gqa, nodes, context, page):
    print(f"tree long fmt={fmt} nkv={nkv} rows={gqa * nodes} context={context} page={page}", flush=True)
    rng, shape, K, V, Q = tree_case(90 + fmt + nodes, fmt, nkv, gqa, 128, nodes, context + nodes)
    _, mask = plain.random_tree(rng, nodes)
    got = run_tree(ws, shape, K, V, split_pages(rng, context + nodes, page), Q, nodes, mask)
    check_tree(shape, K, V, context + nodes, Q, nodes, mask, got)


@pytest.mark.parametrize("fmt,hd", [(Q8, 128), (Q4, 256), (F16, 128)])
def test_tree_padded_rows_and_split(ws, fmt, hd):
    """Rows wider than their heads (their padding never read as keys), and the split-K geometry forced to one and to many chunks."""
    nodes, nkv, gqa, context = 11, 2, 4, 600
    rng, shape, K, V, Q = tree_case(30 + hd, fmt, nkv, gqa, hd, nodes, context + nodes, pad=52)
    _, mask = plain.random_tree(rng, nodes)
    try:
        for groups, wgs in ((0, 0), (1, 1), (19, 300)):
            ws.set_split(groups, wgs)
            print(f"tree padded fmt={fmt} hd={hd} split={groups, wgs}", flush=True)
            got = run_tree(ws, shape, K, V, [300, 311], Q, nodes, mask)
            check_tree(shape, K, V, context + nodes, Q, nodes, mask, got)
    finally:
        ws.set_split(0, 0)


def with_head_gaps(rows, nkv, hb, gap, fill):
    """[n][nkv * hb] bytes with `gap` bytes of `fill` behind every head."""
    h = rows.reshape(-1, nkv, hb)
    return np.concatenate([h, np.full((len(h), nkv, gap), fill, np.uint8)], 2).reshape(len(h), nkv * (hb + gap))


@pytest.mark.parametrize("fmt", [Q8, Q4, F16])
@pytest.mark.parametrize("hd", [128, 256])
def test_heads_with_gaps(ws, fmt, hd):
    """Heads further apart than their bytes (hb): the same tree attention bit for bit as over packed ones, whatever lies between, and the
    same appended heads, with nothing written between."""
    nkv, gqa, nodes, context, gap = 2, 4, 5, 300, 12
    rng, shape, K, V, Q = tree_case(700 + hd + fmt, fmt, nkv, gqa, hd, nodes, context + nodes)
    _, mask = plain.random_tree(rng, nodes)
    wide = bb.Shape(nkv, shape.rows, hd, fmt, nkv * (shape.hb + gap), shape.hb + gap, 0, shape.scale)
    want = run_tree(ws, shape, K, V, [context + nodes], Q, nodes, mask)
    got = run_tree(ws, wide, *(with_head_gaps(x, nkv, shape.hb, gap, 0x7e).reshape(-1) for x in (K, V)), [context + nodes], Q, nodes, mask)
    assert np.array_equal(got[0], want[0]) and np.array_equal(got[1], want[1])
    x = rng.standard_normal((9, (nkv * gqa + 2 * nkv) * hd)).astype(np.float32)
    args = {"w": [None, None], "freq": np.ones(hd // 2, np.float32), "eps": 0.0, "n_rot": hd, "interleaved": False}
    packed, spaced = (gpu_append(bb.Shape(nkv, gqa * 9, hd, fmt, s.rs, s.hb, 0, 1.0), 2, 8, 3, args, x, np.arange(9), 9, gqa, bb.TYPE_F32)
                      for s in (shape, wide))
    assert np.array_equal(packed[0], spaced[0])
    for p, s in zip(packed[1:], spaced[1:]):
        assert np.array_equal(with_head_gaps(p, nkv, shape.hb, gap, 0xa5), s.reshape(-1, wide.rs))


@pytest.mark.parametrize("fmt,nkv,gqa,hd,nodes,context,wgs", [
    (Q8, 3, 7, 128, 49, 4000, 288), (Q4, 3, 7, 128, 49, 4000, 288), (F16, 3, 7, 128, 49, 4000, 288), (Q8, 3, 7, 256, 49, 4000, 864),
    (Q8, 1, 3, 128, 5, 9000, 100), (Q4, 2, 6, 256, 4, 9000, 200), (F16, 1, 8, 256, 3, 9000, 100),
    (F16, 2, 5, 128, 9, 3000, 80), (Q4, 2, 5, 256, 9, 3000, 80), (Q8, 4, 8, 128, 64, 3000, 800)])
def test_tree_rows_and_slots(ws, fmt, nkv, gqa, hd, nodes, context, wgs):
    """Few and many rows with few and many split-K slots: every number of waves per row in the last step, odd numbers of rows among them."""
    print(f"tree rows fmt={fmt} hd={hd} rows={nkv * gqa * nodes} context={context} workgroups={wgs}", flush=True)
    rng, shape, K, V, Q = tree_case(hd + nodes + fmt, fmt, nkv, gqa, hd, nodes, context + nodes)
    _, mask = plain.random_tree(rng, nodes)
    ws.set_split(0, wgs)
    try:
        check_tree(shape, K, V, context + nodes, Q, nodes, mask, run_tree(ws, shape, K, V, [context + nodes], Q, nodes, mask))
    finally:
        ws.set_split(0, 0)


def test_tree_own_stream_repeats(ws):
    """A stream of the caller's, and the same call again: the same bits."""
    rng, shape, K, V, Q = tree_case(31, Q8, 8, 8, 128, 20, 3000)
    _, mask = plain.random_tree(rng, 20)
    st = bb.synth().pa_synth_stream_new()
    a = run_tree(ws, shape, K, V, [1024, 1024, 952], Q, 20, mask, st)
    b = run_tree(ws, shape, K, V, [1024, 1024, 952], Q, 20, mask)
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])
    check_tree(shape, K, V, 3000, Q, 20, mask, a)


def test_tree_offsets_past_32_bits(ws):
    """One page of rows 32 MB apart, 6.7 GB of it: the context's and the tree's rows lie past 32 bits of offset; a rope append
    writes there, and a copy moves rows there."""
    nkv, gqa, hd, nodes, n, rs = 2, 4, 128, 9, 200, 1 << 25
    rng, small, K, V, Q = tree_case(33, Q8, nkv, gqa, hd, nodes, n)
    shape = bb.make_shape(nkv, gqa * nodes, hd, Q8, rs=rs)
    _, mask = plain.random_tree(rng, nodes)
    k, v = bb.DeviceBuffer((n - 1) * rs + small.rs), bb.DeviceBuffer((n - 1) * rs + small.rs)
    dq, dm = buf(Q), buf(mask)
    do, dl = bb.DeviceBuffer(nkv * gqa * nodes * hd * 2), bb.DeviceBuffer(nkv * gqa * nodes * 4)
    put = lambda b, rows, j: b.upload(rows[j * small.rs:(j + 1) * small.rs], j * rs)  # noqa: E731
    get = lambda b, j: b.download(np.uint8, small.rs, j * rs)  # noqa: E731
    try:
        print("tree past 32 bits", flush=True)
        for j in range(n):
            put(k, K, j); put(v, V, j)
        pages = bb.Pages([k.ptr], [v.ptr], [n], [])
        ws.attn_tree(shape, pages, nodes, dm.ptr, dq.ptr, do.ptr, dl.ptr)
        bb.device_sync()
        got = (do.download(np.uint16).reshape(-1, hd), dl.download(np.float32))
        check_tree(small, K, V, n, Q, nodes, mask, got)
        table = bb.LayerTable([pages])
        bb.copy_rows(shape, table, table, n, [191, 193, 198], 191)
        bb.device_sync()
        for X, b in ((K, k), (V, v)):
            for at, j in ((191, 191), (192, 193), (193, 198), (194, 194), (199, 199)):
                assert np.array_equal(get(b, at), X[j * small.rs:(j + 1) * small.rs])
        x = rng.standard_normal((2, 2 * nkv * hd)).astype(np.float32)
        dx, dp = buf(x), buf(np.arange(2, dtype=np.int32))
        rope = bb.make_rope(None, None, 0.0, None, 0, k_stride=2 * nkv * hd, v_stride=2 * nkv * hd)
        bb.append_rope(bb.make_shape(nkv, 0, hd, Q8, rs=rs), pages, n, 197, rope, None, dx.ptr, dx.ptr + 4 * nkv * hd, dp.ptr, 2, None)
        bb.device_sync()
        for t, b in ((0, k), (1, v)):
            vals = np.ascontiguousarray(x.reshape(2, 2, nkv, hd)[:, t])
            want = orc.rows_from_f32(Q8, vals, small.rs, small.hb)
            assert np.array_equal(np.concatenate([get(b, 197), get(b, 198)]), want)
        dx.close(); dp.close()
    finally:
        for b in (k, v, dq, dm, do, dl):
            b.close()


# ---------------------------------------------------------------- norm, rotation and append
def to_type(x, type):
    """fp32 as the bytes of `type`, and the values these hold."""
    if type == bb.TYPE_F32:
        return x, x
    if type == bb.TYPE_F16:
        h = x.astype(np.float16)
        return h, h.astype(np.float32)
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    h = ((u + 0x7fff + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return h, (h.astype(np.uint32) << 16).view(np.float32)


ROPES = [
    # fmt, type, nkv, gqa, hd, n_rot, interleaved, n, pos0, page_keys, position
    (Q8, "f32", 8, 8, 128, 128, False, 1, 0, 64, 0), (Q8, "bf16", 2, 8, 128, 128, False, 37, 50, 64, 131000),
    (Q4, "f16", 4, 6, 256, 64, False, 26, 60, 64, 1000), (F16, "f32", 2, 7, 128, 64, True, 70, 3, 16, 999990),
    (Q8, "f32", 1, 1, 256, 256, True, 5, 0, 5, 16777000), (Q4, "bf16", 3, 2, 128, 32, False, 300, 10, 7, 0),
    (Q8, "f16", 2, 5, 128, 0, False, 9, 1, 64, 4), (F16, "bf16", 2, 1, 256, 130, False, 9, 1, 64, 4), (Q8, "f32", 2, 3, 128, 2, True, 3, 0, 64, 77),
]


def gpu_append(shape, n_pages, page_keys, pos0, rope_args, qkv, pos, n, gqa, type, poison=0xa5):
    """The page bytes (K, V) and q_out of an append from one fused [n][width] buffer; pages start poisoned."""
    nkv, hd = shape.nkv, shape.hd
    w, f = rope_args["w"], rope_args["freq"]
    dw = [buf(x) if x is not None else None for x in w]
    df, dp, dx = buf(f if f.size else np.zeros(1, np.float32)), buf(pos.astype(np.int32)), buf(qkv)
    size = {bb.TYPE_F32: 4}.get(type, 2)
    pages = bb.alloc_pages(n_pages, page_keys * shape.rs)
    dq = buf(np.full(nkv * gqa * n * hd + 8, 3.5, np.float32))
    try:
        for b in pages.bufs:
            b.upload(np.full(page_keys * shape.rs, poison, np.uint8))
        width = qkv.shape[1]
        rope = bb.make_rope(dw[0].ptr if dw[0] else None, dw[1].ptr if dw[1] else None, rope_args["eps"], df.ptr, rope_args["n_rot"],
                            rope_args["interleaved"], type, width, width, width)
        lead = rope_args.get("lead", 0)
        at = [dx.ptr + size * (lead + hd * i) for i in (0, nkv * gqa, nkv * gqa + nkv)]
        bb.append_rope(shape, pages, page_keys, pos0, rope, at[0] if gqa else None, at[1], at[2], dp.ptr, n, dq.ptr if gqa else None)
        bb.device_sync()
        q = dq.download(np.float32)
        assert np.all(q[nkv * gqa * n * hd:] == 3.5)
        k, v = (np.concatenate([pages.bufs[2 * i + t].download(np.uint8, page_keys * shape.rs) for i in range(n_pages)]) for t in (0, 1))
        return q[:nkv * gqa * n * hd].reshape(nkv, gqa, n, hd), k, v
    finally:
        pages.close()
        for b in [*dw, df, dp, dx, dq]:
            if b:
                b.close()


@pytest.mark.parametrize("fmt,type,nkv,gqa,hd,n_rot,interleaved,n,pos0,page_keys,position", ROPES)
@pytest.mark.parametrize("norm", [True, False])
def test_append_rope(fmt, type, nkv, gqa, hd, n_rot, interleaved, n, pos0, page_keys, position, norm):
    print(f"append_rope fmt={fmt} {type} nkv={nkv} gqa={gqa} hd={hd} rot={n_rot} {interleaved} n={n} norm={norm}", flush=True)
    type = {"f32": bb.TYPE_F32, "f16": bb.TYPE_F16, "bf16": bb.TYPE_BF16}[type]
    rng = np.random.default_rng(n + hd + n_rot)
    heads = nkv * gqa + 2 * nkv
    lead, width = (1, heads * hd + 5) if type == bb.TYPE_F32 else (2, heads * hd + 6)   # the heads inside wider rows
    x = (rng.standard_normal((n, width)) * rng.choice([1e-3, 1.0, 30.0], (n, 1))).astype(np.float32)
    raw, vals = to_type(x, type)
    vals = vals[:, lead:lead + heads * hd].reshape(n, heads, hd)
    w = [(1.0 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)] if norm else [None, None]
    freq = (1e6 ** (-2.0 * np.arange(n_rot // 2) / max(n_rot, 1))).astype(np.float32)
    pos = position + rng.integers(0, 5, n)                            # a tree's: siblings share one
    hb = orc.head_bytes(fmt, hd); rs = nkv * hb + 4
    shape = bb.make_shape(nkv, gqa * n, hd, fmt, rs=rs)
    n_pages = (pos0 + n + page_keys - 1) // page_keys + 1
    q, k, v = gpu_append(shape, n_pages, page_keys, pos0, {"w": w, "freq": freq, "eps": 1e-5, "n_rot": n_rot, "interleaved": interleaved,
                                                          "lead": lead}, raw, pos, n, gqa, type)
    nq = nkv * gqa
    wq = plain.norm_rope(vals[:, :nq], w[0], 1e-5, freq, pos, n_rot, interleaved)
    wk = plain.norm_rope(vals[:, nq:nq + nkv], w[1], 1e-5, freq, pos, n_rot, interleaved)
    # fp64 rounded once to fp32: half a step, and what fp64 itself loses (a pair's two terms may cancel, 2^-50 of their size)
    size = np.abs(wq).max(2, keepdims=True)
    got = q.transpose(2, 0, 1, 3).reshape(n, nq, hd)
    assert np.all(np.abs(got - wq) <= 2.0 ** -24 * np.abs(wq) + 2.0 ** -49 * size)
    want = np.full((n_pages * page_keys, rs), 0xa5, np.uint8)
    for got, vals3 in ((k, wk.astype(np.float32)), (v, vals[:, nq + nkv:])):
        rows = orc.rows_from_f32(fmt, np.ascontiguousarray(vals3), rs, hb).reshape(n, rs)
        want[pos0:pos0 + n, :nkv * hb] = rows[:, :nkv * hb]
        assert np.array_equal(got.reshape(-1, rs), want)              # the new rows, and not a byte beside them


def test_append_rope_keys_only_and_values_of_zero():
    """No queries; heads of zeros (the norm divides by sqrt(eps), the quantizer by nothing)."""
    nkv, hd, n = 2, 128, 3
    x = np.zeros((n, 2 * nkv * hd), np.float32)
    x[1] = np.random.default_rng(3).standard_normal(2 * nkv * hd)
    shape = bb.make_shape(nkv, 0, hd, Q8)
    w = np.ones(hd, np.float32)
    freq = np.ones(64, np.float32)
    _, k, v = gpu_append(shape, 1, 4, 1, {"w": [w, w], "freq": freq, "eps": 1e-6, "n_rot": 128, "interleaved": False}, x, np.arange(3), n, 0,
                         bb.TYPE_F32)
    vals = x.reshape(n, 2 * nkv, hd)
    for got, ref in ((k, plain.norm_rope(vals[:, :nkv], w, 1e-6, freq, np.arange(3), 128, False).astype(np.float32)), (v, vals[:, nkv:])):
        rows = orc.rows_from_f32(Q8, np.ascontiguousarray(ref), shape.rs, shape.hb).reshape(n, -1)
        assert np.array_equal(got.reshape(4, -1)[1:], rows) and np.all(got.reshape(4, -1)[0] == 0xa5)


def test_append_rope_many_tokens_and_positions_before_zero():
    """More tokens than a launch takes (65,535), over more pages than one names (16); negative positions turn the other way."""
    nkv, gqa, hd, n, pos0, page_keys = 1, 1, 128, 70000, 11, 2048
    rng = np.random.default_rng(5)
    x = rng.standard_normal((n, 3 * hd)).astype(np.float32)
    pos = rng.integers(-1000, 140000, n)
    freq = (1e4 ** (-2.0 * np.arange(64) / 128)).astype(np.float32)
    w = [(1.0 + 0.3 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
    shape = bb.make_shape(nkv, gqa * n, hd, Q4)
    n_pages = (pos0 + n + page_keys - 1) // page_keys
    q, k, v = gpu_append(shape, n_pages, page_keys, pos0, {"w": w, "freq": freq, "eps": 1e-6, "n_rot": 128, "interleaved": False}, x, pos, n, gqa,
                         bb.TYPE_F32)
    vals = x.reshape(n, 3, hd)
    wq, wk = (plain.norm_rope(vals[:, i:i + 1], w[i], 1e-6, freq, pos, 128, False) for i in (0, 1))
    assert np.all(np.abs(q[0, 0] - wq[:, 0]) <= 2.0 ** -24 * np.abs(wq[:, 0]) + 2.0 ** -49 * np.abs(wq).max(2))
    for got, ref in ((k, wk.astype(np.float32)), (v, vals[:, 2:])):
        rows = orc.rows_from_f32(Q4, np.ascontiguousarray(ref), shape.rs, shape.hb).reshape(n, -1)
        assert np.array_equal(got.reshape(-1, shape.rs)[pos0:pos0 + n], rows)


# ---------------------------------------------------------------- log probabilities
def gpu_logprobs(ws, raw, type, vocab, scale, given, n_top, stream=None, wanted=True):
    rows, stride = raw.shape
    dx, dg = buf(raw), buf(np.ascontiguousarray(given, np.int32) if given.size else np.zeros(1, np.int32))
    ng = given.shape[1]
    out = [buf(np.full(max(1, rows * c) + 3, 9.0, np.float32)) for c in (ng, 1, 1, n_top)]
    ids = buf(np.full(max(1, rows * n_top) + 3, 99, np.int32))
    try:
        ws.logprobs(dx.ptr, type, rows, vocab, stride, scale, dg.ptr, ng, n_top, out[0].ptr, out[1].ptr if wanted else None,
                    out[2].ptr if wanted else None, ids.ptr, out[3].ptr, stream)
        bb.device_sync()
        f = [o.download(np.float32) for o in out]
        i = ids.download(np.int32)
        for a, c in zip(f, (ng, 1, 1, n_top)):
            assert np.all(a[rows * c:] == 9.0)
        assert np.all(i[rows * n_top:] == 99)
        return (f[0][:rows * ng].reshape(rows, ng), f[1][:rows], f[2][:rows], i[:rows * n_top].reshape(rows, n_top),
                f[3][:rows * n_top].reshape(rows, n_top))
    finally:
        for b in (dx, dg, ids, *out):
            b.close()


def check_logprobs(x, scale, given, n_top, got):
    """An exponent's argument scale (x - m) is off by 2^-23 of itself (two roundings), e^ by 2^-23, and the sums, 64 values of a
    thread and at most 24 joins, by 90 half steps: S is off by its terms' share of these, at most (30 + 2 + 90) 2^-24 where
    only terms above e^-15 matter (the others' sizes cover their larger share), under 2^-17; ln S as much absolutely, T / S as much
    of its own size and, from the weights, of ln S's."""
    logp, lse, ent, top, top_lp = plain.logprobs(x, scale, given, n_top)
    y = np.where(np.isfinite(x), np.abs(x * scale), 0.0).max(1)
    big = 2.0 ** -17 + 2.0 ** -22 * (y + np.where(np.isfinite(lse), np.abs(lse), 0.0))
    for g, w, tol in ((got[0], logp, big[:, None]), (got[1], lse, big), (got[2], ent, 2.0 ** -17 * (2 + np.abs(ent))), (got[4], top_lp, big[:, None])):
        assert np.array_equal(np.isnan(g), np.isnan(w)) and np.array_equal(np.isneginf(g), np.isneginf(w))
        ok = np.isfinite(w)
        assert np.all(np.isfinite(g[ok]))
        assert np.all(np.abs(g - w)[ok] <= np.broadcast_to(tol, w.shape)[ok])
    assert np.array_equal(got[3], top)


@pytest.mark.parametrize("type", [bb.TYPE_F32, bb.TYPE_F16, bb.TYPE_BF16])
@pytest.mark.parametrize("rows,vocab,stride,n_given,n_top", [
    (1, 1, 1, 1, 1), (2, 3, 3, 2, 5), (5, 255, 257, 3, 32), (3, 4096, 4096, 1, 20), (4, 4097, 4099, 0, 7), (1, 151936, 151936, 4, 32),
    (17, 50001, 50001, 3, 8), (2, 16385, 20000, 300, 1), (9, 32000, 32000, 1, 0), (130, 40000, 40001, 1, 5), (300, 1000, 1000, 2, 32),
    (1, 1000003, 1000003, 2, 32)])
def test_logprobs(ws, type, rows, vocab, stride, n_given, n_top):
    print(f"logprobs type={type} rows={rows} vocab={vocab} stride={stride} given={n_given} top={n_top}", flush=True)
    rng = np.random.default_rng(rows + vocab)
    x = (rng.standard_normal((rows, stride)) * 2.5).astype(np.float32)
    x[:, vocab:] = 1e9                                                # the padding must not count
    x[np.arange(rows), rng.integers(0, vocab, rows)] += (rng.random(rows) * 25).astype(np.float32)
    x[:, rng.integers(0, vocab, max(1, vocab // 100))] = -np.inf
    x[-1, 0] = 3.0
    raw, vals = to_type(x, type)
    given = rng.integers(0, vocab, (rows, n_given)).astype(np.int32)
    if n_given > 1:
        given[0, 0], given[-1, 1] = -1, vocab
    for scale in (1.0, 0.7):
        check_logprobs(vals[:, :vocab], scale, given, n_top, gpu_logprobs(ws, raw, type, vocab, scale, given, n_top))


@pytest.mark.parametrize("type", [bb.TYPE_F32, bb.TYPE_BF16])
@pytest.mark.parametrize("n_top", [1, 5, 32])
def test_logprobs_whole_rows_of_a_workgroup(ws, type, n_top):
    """So many rows that a workgroup streams a whole one: values in ascending, descending and random order, with few different values
    (ties, the lowest id first), ever larger towards one lane's places, and the best ones at the row's end."""
    rows, vocab = 1026, 9001
    print(f"logprobs whole rows type={type} top={n_top}", flush=True)
    rng = np.random.default_rng(n_top)
    x = (rng.standard_normal((rows, vocab)) * 2.0).astype(np.float32)
    up = np.linspace(-9.0, 9.0, vocab, dtype=np.float32)
    x[0::6], x[1::6] = up, up[::-1]
    x[2::6] = rng.integers(-3, 4, x[2::6].shape)
    x[3::6, 5::1024] += np.arange(len(range(5, vocab, 1024)), dtype=np.float32) + 9.0
    x[4::6, -40:] += 12.0
    raw, vals = to_type(x, type)
    given = rng.integers(0, vocab, (rows, 1)).astype(np.int32)
    check_logprobs(vals, 1.0, given, n_top, gpu_logprobs(ws, raw, type, vocab, 1.0, given, n_top))


@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_logprobs_edges(ws, vocab):
    """Rows of equal values, of -inf only, of a few finite values among -inf, of +inf, of NaN, of ascending and of descending values,
    of the lowest and the largest floats, of +0 and -0, all the best values in one thread's share."""
    rng = np.random.default_rng(vocab)
    big = np.finfo(np.float32).max
    r = [np.zeros(vocab), np.full(vocab, -np.inf), np.full(vocab, -np.inf), rng.standard_normal(vocab), rng.standard_normal(vocab),
         np.arange(vocab) * 1e-3, -np.arange(vocab) * 1e-3, np.full(vocab, -big), rng.standard_normal(vocab), np.where(np.arange(vocab) % 2, 0.0, -0.0),
         rng.standard_normal(vocab), np.full(vocab, -1e30), np.full(vocab, 60000.0)]
    x = np.array(r, np.float32)
    x[2, [7, 31, vocab - 1]] = [1.0, 2.0, 1.0]
    x[3, vocab // 2] = np.inf
    x[4, [3, vocab - 2]] = [np.nan, -np.nan]
    x[8, 5] = big
    x[10, 11::256] = 50.0 + rng.random(len(x[10, 11::256]))
    given = np.tile(np.array([[0, 7, vocab - 1, vocab // 2, 3, 5, 11]], np.int32), (len(r), 1))
    print(f"logprobs edges vocab={vocab}", flush=True)
    for n_top in (1, 5, 32):
        check_logprobs(x, 1.0, given, n_top, gpu_logprobs(ws, x, bb.TYPE_F32, vocab, 1.0, given, n_top))


def test_logprobs_best_in_few_places(ws):
    """The best in every other 4,096 values only (the join's lists then hold them in half of the lanes), all in one thread's share,
    and in ascending and descending runs of the whole row."""
    rng = np.random.default_rng(5)
    vocab = 38 * 4096 - 7
    x = rng.standard_normal((4, vocab)).astype(np.float32)
    x[0] += np.where(np.arange(vocab) // 4096 % 2 == 0, 100.0, 0.0).astype(np.float32)
    x[1, 20::1024] += 50.0
    x[2] = np.sort(x[2])
    x[3] = np.sort(x[3])[::-1]
    given = rng.integers(0, vocab, (4, 1)).astype(np.int32)
    print("logprobs few places", flush=True)
    for rows in ([0], [1], [2], [3], [0, 1, 2, 3]):
        for n_top in (32, 31, 3):
            check_logprobs(x[rows], 1.0, given[rows], n_top, gpu_logprobs(ws, x[rows], bb.TYPE_F32, vocab, 1.0, given[rows], n_top))


def test_logprobs_largest_vocabulary(ws):
    vocab = 1 << 24
    rng = np.random.default_rng(6)
    x = rng.standard_normal((1, vocab)).astype(np.float32)
    best = rng.choice(vocab, 32, replace=False)
    x[0, best] = 10.0 + np.arange(32) / 4
    print("logprobs 2^24", flush=True)
    got = gpu_logprobs(ws, x, bb.TYPE_F32, vocab, 1.0, np.array([[best[3]]], np.int32), 32)
    y = x.astype(np.float64)
    lse = 0.0 + np.log(np.exp(y).sum())
    assert abs(got[1][0] - lse) < 2.0 ** -17 + 2.0 ** -22 * 40        # as check_logprobs counts it
    assert np.array_equal(got[3][0], best[::-1]) and abs(got[0][0, 0] - (x[0, best[3]] - lse)) < 2.0 ** -16
    lp = y - lse
    assert abs(got[2][0] + (np.exp(lp) * lp).sum()) < 2.0 ** -17 * 20


def test_logprobs_wanted_only(ws):
    rng = np.random.default_rng(1)
    x = rng.standard_normal((3, 700)).astype(np.float32)
    given = rng.integers(0, 700, (3, 2)).astype(np.int32)
    got = gpu_logprobs(ws, x, bb.TYPE_F32, 700, 1.0, given, 3, wanted=False)
    assert np.all(got[1] == 9.0) and np.all(got[2] == 9.0)
    full = gpu_logprobs(ws, x, bb.TYPE_F32, 700, 1.0, given, 3)
    assert np.array_equal(got[0], full[0]) and np.array_equal(got[3], full[3]) and np.array_equal(got[4], full[4])


def test_two_streams_at_once():
    """Two workspaces on two streams, their calls in flight together: the results of one after the other."""
    syn = bb.synth()
    st = [syn.pa_synth_stream_new() for _ in range(2)]
    w = [bb.Workspace() for _ in range(2)]
    loops = [Loop(21 + i, Q8, 128, 700, 12, vocab=50000) for i in range(2)]
    print("two streams", flush=True)
    try:
        for l in loops:
            l.append(l.d["x0"], l.d["pos0"], l.context, 0, None, None)
            l.new_tree()
        bb.device_sync()
        want = []
        for i, l in enumerate(loops):
            l.step(w[i], st[i])
            bb.device_sync()
            want.append(l.outputs())
        for _ in range(5):
            for l in loops:
                for k in ("o", "lse", "lp", "top"):
                    l.d[k].upload(np.full(l.d[k].nbytes, 0x5a, np.uint8))
            for _ in range(4):
                for i, l in enumerate(loops):
                    l.step(w[i], st[i])
            bb.device_sync()
            for l, o in zip(loops, want):
                got = l.outputs()
                assert all(np.array_equal(got[k], o[k]) for k in o)
    finally:
        for l in loops:
            l.close()
        for a in w:
            a.close()


# ---------------------------------------------------------------- row copies
class Cache:
    """Random pages of `layers` layers, on the device and here."""

    def __init__(self, rng, layers, n_pages, page_keys, rs, skew=0):
        self.rs, self.page_keys, self.skew = rs, page_keys, skew
        self.bytes = rng.integers(0, 256, (layers, 2, n_pages * page_keys, rs), dtype=np.uint8)
        nb = page_keys * rs
        self.buf = bb.DeviceBuffer(layers * 2 * n_pages * (nb + 16) + 16)
        self.table, at = [], self.buf.ptr + skew
        self.at = {}
        for l in range(layers):
            ptr = []
            for t in range(2):
                for p in range(n_pages):
                    self.at[l, t, p] = at - self.buf.ptr
                    self.buf.upload(self.bytes[l, t, p * page_keys:(p + 1) * page_keys].reshape(-1), at - self.buf.ptr)
                    ptr.append(at)
                    at += (nb + 15) // 16 * 16
            self.table.append(bb.Pages(ptr[:n_pages], ptr[n_pages:], [page_keys] * n_pages, []))
        self.table = bb.LayerTable(self.table)

    def now(self):
        got = np.empty_like(self.bytes)
        for (l, t, p), at in self.at.items():
            n = self.page_keys * self.rs
            got[l, t, p * self.page_keys:(p + 1) * self.page_keys] = self.buf.download(np.uint8, n, at).reshape(-1, self.rs)
        return got


def copied(src, dst, at, to, row):
    want = dst.copy()
    want[:, :, to:to + len(at), :row] = src[:, :, list(at), :row]
    return want


@pytest.mark.parametrize("fmt,nkv,hd,pad,skew", [(Q8, 8, 128, 0, 0), (Q4, 1, 128, 0, 0), (Q8, 3, 128, 10, 2), (F16, 2, 256, 16, 0), (Q4, 1, 128, 1, 1)])
@pytest.mark.parametrize("layers,page_keys,n_pages,at,to", [
    (1, 64, 1, [5], 5), (3, 64, 2, [5, 6, 9, 60], 4), (2, 16, 4, list(range(7, 60, 2)), 7), (70, 32, 2, [30, 31, 40, 63], 30),
    (2, 100, 3, list(range(1, 300)), 0), (2, 100, 3, sorted(set(range(20, 300)) - {21, 150}), 11), (1, 7, 20, range(40, 140), 3),
    (2, 64, 3, range(100, 150), 20), (2, 64, 1, range(3, 64), 3)])
def test_copy_rows_in_place(fmt, nkv, hd, pad, skew, layers, page_keys, n_pages, at, to):
    print(f"copy in place fmt={fmt} nkv={nkv} pad={pad} skew={skew} layers={layers} page={page_keys} n={len(at)}", flush=True)
    rng = np.random.default_rng(len(at) + to)
    rs = nkv * orc.head_bytes(fmt, hd) + pad
    shape = bb.make_shape(nkv, 1, hd, fmt, rs=rs)
    c = Cache(rng, layers, n_pages, page_keys, rs, skew)
    bb.copy_rows(shape, c.table, c.table, page_keys, at, to)
    bb.device_sync()
    assert np.array_equal(c.now(), copied(c.bytes, c.bytes, at, to, nkv * shape.hb))
    c.buf.close()


@pytest.mark.parametrize("fmt,nkv,hd,pad,skew", [(Q8, 8, 128, 0, 0), (Q4, 1, 128, 0, 0), (Q8, 3, 128, 10, 2), (F16, 2, 256, 16, 0), (Q4, 1, 128, 1, 1)])
@pytest.mark.parametrize("layers,page_keys,at,to", [
    (1, 64, range(0, 1), 0), (3, 64, range(0, 64), 0), (66, 64, range(3, 60), 3), (2, 50, range(0, 150), 0), (2, 50, range(17, 120), 31),
    (2, 50, [1, 2, 3, 70, 149], 99), (1, 1000, range(0, 2500), 300), (2, 50, list(range(10, 130)), 0)])
def test_copy_rows_fork(fmt, nkv, hd, pad, skew, layers, page_keys, at, to):
    print(f"copy fork fmt={fmt} nkv={nkv} pad={pad} skew={skew} layers={layers} page={page_keys} n={len(at)}", flush=True)
    rng = np.random.default_rng(len(at) + to)
    rs = nkv * orc.head_bytes(fmt, hd) + pad
    shape = bb.make_shape(nkv, 1, hd, fmt, rs=rs)
    a, b = Cache(rng, layers, 3, page_keys, rs, skew), Cache(rng, layers, 3, page_keys, rs)
    bb.copy_rows(shape, a.table, b.table, page_keys, at, to)
    bb.device_sync()
    assert np.array_equal(a.now(), a.bytes)
    assert np.array_equal(b.now(), copied(a.bytes, b.bytes, at, to, nkv * shape.hb))
    a.buf.close(); b.buf.close()


@pytest.mark.parametrize("layers,at,to,shared", [
    (2, range(0, 120), 0, {0, 1}), (3, range(10, 64), 10, {0}), (2, [5, 6, 7, 60, 130], 5, {0, 2}), (2, list(range(50, 140)), 50, {1}),
    (2, range(100, 140), 4, {0})])
def test_copy_rows_into_a_table_that_shares_pages(layers, at, to, shared):
    """A fork whose table holds its parent's own full pages (in every layer, and in one layer only) and copies of the others: rows of a
    shared page move within it or stay, rows that stay in position still reach the pages of its own."""
    print(f"copy shared={shared} layers={layers} n={len(at)} to={to}", flush=True)
    rng = np.random.default_rng(len(at))
    shape = bb.make_shape(2, 1, 128, Q8)
    for where in (range(layers), range(1)):                          # the layers that share them
        a, b = Cache(rng, layers, 3, 50, shape.rs), Cache(rng, layers, 3, 50, shape.rs)
        share = lambda l, p: l in where and p in shared
        table = [bb.Pages([(a if share(l, p) else b).table.k[3 * l + p] for p in range(3)],
                          [(a if share(l, p) else b).table.v[3 * l + p] for p in range(3)], [50] * 3, []) for l in range(layers)]
        want_a, want_b = a.bytes.copy(), b.bytes.copy()
        for l in range(layers):
            for i, f in enumerate(at):
                (want_a if share(l, (to + i) // 50) else want_b)[l, :, to + i] = a.bytes[l, :, f]
        bb.copy_rows(shape, a.table, bb.LayerTable(table), 50, at, to)
        bb.device_sync()
        assert np.array_equal(a.now(), want_a) and np.array_equal(b.now(), want_b)
        a.buf.close(); b.buf.close()


# ---------------------------------------------------------------- the loop
class Loop:
    """A toy model of one layer whose next-token logits come from the tree attention's rows: append the tree's tokens, attend, score."""

    def __init__(self, seed, fmt, hd, context, nodes, page_keys=64, nkv=2, gqa=4, vocab=3001):
        rng = np.random.default_rng(seed)
        self.rng, self.fmt, self.hd, self.nkv, self.gqa, self.nodes, self.context, self.page_keys, self.vocab = rng, fmt, hd, nkv, gqa, nodes, context, \
            page_keys, vocab
        self.heads = nkv * gqa + 2 * nkv
        self.n_pages = (context + nodes + page_keys - 1) // page_keys
        self.shape = bb.make_shape(nkv, gqa * nodes, hd, fmt)
        self.freq = (1e4 ** (-2.0 * np.arange(hd // 2) / hd)).astype(np.float32)
        self.w = [(1.0 + 0.2 * rng.standard_normal(hd)).astype(np.float32) for _ in range(2)]
        self.x0 = rng.standard_normal((context, self.heads * hd)).astype(np.float32)
        self.pages = bb.alloc_pages(self.n_pages, page_keys * self.shape.rs)
        for b in self.pages.bufs:
            b.upload(np.zeros(page_keys * self.shape.rs, np.uint8))
        n = context + nodes
        self.pages.nkeys = [min(page_keys, n - i * page_keys) for i in range(self.n_pages)]
        self.d = {k: buf(v) for k, v in dict(w0=self.w[0], w1=self.w[1], freq=self.freq, x0=self.x0, pos0=np.arange(context, dtype=np.int32),
                                             x=np.zeros((nodes, self.heads * hd), np.float32), pos=np.zeros(nodes, np.int32),
                                             mask=np.zeros(nodes, np.uint64), q=np.zeros((nkv * gqa * nodes, hd), np.float32),
                                             logits=np.zeros((nodes, vocab), np.float32), ids=np.zeros((nodes, 2), np.int32),
                                             o=np.zeros((nkv * gqa * nodes, hd), np.uint16), lse=np.zeros(nkv * gqa * nodes, np.float32),
                                             lp=np.zeros(nodes * (2 + 1 + 1 + 4), np.float32), top=np.zeros(nodes * 4, np.int32)).items()}

    def append(self, x, pos, n, at, q, st):
        rope = bb.make_rope(self.d["w0"].ptr, self.d["w1"].ptr, 1e-6, self.d["freq"].ptr, self.hd, False, bb.TYPE_F32, self.heads * self.hd,
                            self.heads * self.hd, self.heads * self.hd)
        e = [x.ptr + 4 * self.hd * i for i in (0, self.nkv * self.gqa, self.nkv * self.gqa + self.nkv)]
        shape = bb.make_shape(self.nkv, self.gqa * n if q else 0, self.hd, self.fmt)
        bb.append_rope(shape, self.pages, self.page_keys, at, rope, e[0] if q else None, e[1], e[2], pos.ptr, n, q, st)

    def new_tree(self):
        x = self.rng.standard_normal((self.nodes, self.heads * self.hd)).astype(np.float32)
        self.parent, mask = plain.random_tree(self.rng, self.nodes)
        depth = np.zeros(self.nodes, np.int32)
        for i in range(1, self.nodes):
            depth[i] = depth[self.parent[i]] + 1
        logits = (self.rng.standard_normal((self.nodes, self.vocab)) * 3).astype(np.float32)
        ids = self.rng.integers(0, self.vocab, (self.nodes, 2)).astype(np.int32)
        for k, v in dict(x=x, pos=self.context + depth, mask=mask, logits=logits, ids=ids).items():
            self.d[k].upload(v)
        return x, self.context + depth, mask, logits, ids

    def step(self, ws, st):
        d, n = self.d, self.nodes
        self.append(d["x"], d["pos"], n, self.context, d["q"].ptr, st)
        ws.attn_tree(self.shape, self.pages, n, d["mask"].ptr, d["q"].ptr, d["o"].ptr, d["lse"].ptr, st)
        ws.logprobs(d["logits"].ptr, bb.TYPE_F32, n, self.vocab, self.vocab, 0.8, d["ids"].ptr, 2, 4, d["lp"].ptr, d["lp"].ptr + 4 * 2 * n,
                    d["lp"].ptr + 4 * 3 * n, d["top"].ptr, d["lp"].ptr + 4 * 4 * n, st)

    def outputs(self):
        return {k: self.d[k].download(np.uint8) for k in ("q", "o", "lse", "lp", "top")} | {
            "pages": np.concatenate([b.download(np.uint8) for b in self.pages.bufs])}

    def rows(self, t, n):
        """The first n rows of K (t 0) or V (1)."""
        return np.concatenate([b.download(np.uint8) for b in self.pages.bufs[t::2]])[:n * self.shape.rs]

    def check(self, x, pos, mask, logits, ids):
        n, nq = self.context + self.nodes, self.nkv * self.gqa
        vals = x.reshape(self.nodes, self.heads, self.hd)
        q = plain.norm_rope(vals[:, :nq], self.w[0], 1e-6, self.freq, pos, self.hd, False).astype(np.float32)
        k = plain.norm_rope(vals[:, nq:nq + self.nkv], self.w[1], 1e-6, self.freq, pos, self.hd, False).astype(np.float32)
        rs, hb = self.shape.rs, self.shape.hb
        K, V = self.rows(0, n), self.rows(1, n)
        assert np.array_equal(K[self.context * rs:], orc.rows_from_f32(self.fmt, k, rs, hb))
        assert np.array_equal(V[self.context * rs:], orc.rows_from_f32(self.fmt, np.ascontiguousarray(vals[:, nq + self.nkv:]), rs, hb))
        Q = q.reshape(self.nodes, self.nkv, self.gqa, self.hd).transpose(1, 2, 0, 3).reshape(-1, self.hd)
        assert np.array_equal(self.d["q"].download(np.float32).reshape(-1, self.hd), Q)
        rows = self.nkv * self.gqa * self.nodes
        check_tree(self.shape, K, V, n, Q, self.nodes, mask, (self.d["o"].download(np.uint16).reshape(rows, -1), self.d["lse"].download(np.float32)))
        lp, m = self.d["lp"].download(np.float32), self.nodes
        check_logprobs(logits, 0.8, ids, 4, (lp[:2 * m].reshape(m, 2), lp[2 * m:3 * m], lp[3 * m:4 * m],
                                             self.d["top"].download(np.int32).reshape(m, 4), lp[4 * m:].reshape(m, 4)))

    def close(self):
        self.pages.close()
        for b in self.d.values():
            b.close()


@pytest.mark.parametrize("fmt,hd,context,nodes", [(Q8, 128, 150, 13), (Q4, 128, 40, 30), (F16, 256, 100, 9), (Q8, 256, 61, 6)])
def test_loop(ws, fmt, hd, context, nodes):
    """Context and tree appended, the tree attended and scored, an accepted path moved together: the cache then holds, bit for
    bit, what it would hold had the accepted tokens been appended alone, and a fork of its last page the same."""
    print(f"loop fmt={fmt} hd={hd} context={context} nodes={nodes}", flush=True)
    m = Loop(7 + hd + fmt, fmt, hd, context, nodes)
    try:
        m.append(m.d["x0"], m.d["pos0"], context, 0, None, None)
        x, pos, mask, logits, ids = m.new_tree()
        m.step(ws, None)
        bb.device_sync()
        m.check(x, pos, mask, logits, ids)
        path = [j for j in range(nodes) if int(mask[nodes - 1]) >> j & 1]     # the last node's ancestors and itself
        table = bb.LayerTable([m.pages])
        bb.copy_rows(m.shape, table, table, m.page_keys, [context + j for j in path], context)
        alone = Loop(7 + hd + fmt, fmt, hd, context, nodes)
        alone.append(alone.d["x0"], alone.d["pos0"], context, 0, None, None)
        kept = buf(np.ascontiguousarray(x[path])); kpos = buf(np.ascontiguousarray(pos[path].astype(np.int32)))
        alone.append(kept, kpos, len(path), context, None, None)
        bb.device_sync()
        n = context + len(path)
        assert np.array_equal(m.rows(0, n), alone.rows(0, n)) and np.array_equal(m.rows(1, n), alone.rows(1, n))
        fork = bb.alloc_pages(m.n_pages, m.page_keys * m.shape.rs)
        last = (n - 1) // m.page_keys * m.page_keys
        bb.copy_rows(m.shape, table, bb.LayerTable([fork]), m.page_keys, range(last, n), last)
        bb.device_sync()
        for t in (0, 1):
            assert np.array_equal(fork.bufs[2 * (last // m.page_keys) + t].download(np.uint8, (n - last) * m.shape.rs),
                                  m.rows(t, n)[last * m.shape.rs:])
        fork.close(); kept.close(); kpos.close(); alone.close()
    finally:
        m.close()


@pytest.mark.parametrize("fmt,hd,nodes", [(Q8, 128, 16), (F16, 128, 5), (Q4, 256, 7)])
def test_loop_graph(fmt, hd, nodes):
    """The step captured once, replayed over new trees (tokens, masks, logits uploaded between replays) with eager steps of another
    cache on the same workspace in between: every replay gives what an eager step gives, bit for bit. A capture that would have to
    grow the workspace is refused."""
    print(f"loop graph fmt={fmt} hd={hd} nodes={nodes}", flush=True)
    syn = bb.synth()
    w = bb.Workspace()
    st = syn.pa_synth_stream_new()
    m, other = Loop(11 + hd, fmt, hd, 130, nodes), Loop(12 + hd, fmt, hd, 200, nodes)
    gx = None
    try:
        for l in (m, other):
            l.append(l.d["x0"], l.d["pos0"], l.context, 0, None, st)
            l.new_tree()
        assert syn.pa_synth_capture_begin(st) == 0
        with pytest.raises(bb.PaHipError, match="must grow"):
            w.attn_tree(m.shape, m.pages, nodes, m.d["mask"].ptr, m.d["q"].ptr, m.d["o"].ptr, m.d["lse"].ptr, st)
        g = syn.pa_synth_capture_end(st)
        if g:
            syn.pa_synth_graph_free(g)
        other.step(w, st)
        m.step(w, st)
        assert syn.pa_synth_stream_sync(st) == 0
        assert syn.pa_synth_capture_begin(st) == 0
        m.step(w, st)
        gx = syn.pa_synth_capture_end(st)
        assert gx, "capture failed"
        for rep in range(4):
            tree = m.new_tree()
            assert syn.pa_synth_graph_launch(gx, st) == 0
            assert syn.pa_synth_stream_sync(st) == 0
            got = m.outputs()
            m.check(*tree)
            for k in ("o", "lse", "lp", "top", "q"):
                m.d[k].upload(np.full(m.d[k].nbytes, 0x5a, np.uint8))
            m.step(w, st)
            other.new_tree()
            other.step(w, st)
            assert syn.pa_synth_stream_sync(st) == 0
            want = m.outputs()
            for k in want:
                assert np.array_equal(got[k], want[k]), f"replay {rep}: {k}"
    finally:
        if gx:
            syn.pa_synth_graph_free(gx)
        w.close()
        m.close()
        other.close()
