"""What pa_hip_attn_tree, pa_hip_logprobs, pa_hip_append_rope and pa_hip_copy_rows refuse, on the CPU: every refusal comes before
any work is enqueued, so none needs a device (the pointers here are numbers that nothing may follow)."""
import ctypes as C

import pytest

import backburner_amd as bb

P = 0x10000                                              # a 16-byte aligned "device pointer"


def refused(what, call):
    with pytest.raises(bb.PaHipError) as e:
        call()
    assert what in str(e.value), str(e.value)


class NoWorkspace(bb.Workspace):
    def __init__(self):
        self.ptr = None


def pages(counts, k=P, v=P):
    return bb.Pages([k] * len(counts), [v] * len(counts), list(counts), [])


# ---------------------------------------------------------------- tree attention
def tree(shape=None, counts=(100, 50), n_nodes=4, mask=P, Q=P, Oh=P, lse=P, k=P, v=P):
    shape = shape or bb.make_shape(2, 16, 128, bb.FMT_Q8_0)
    NoWorkspace().attn_tree(shape, pages(counts, k, v), n_nodes, mask, Q, Oh, lse)


@pytest.mark.parametrize("what,kw", [
    ("n_nodes must be 1..64", dict(n_nodes=0)),
    ("n_nodes must be 1..64", dict(n_nodes=65, shape=bb.make_shape(2, 65, 128, bb.FMT_Q8_0))),
    ("multiple of n_nodes", dict(n_nodes=5)),
    ("qmode must be 0", dict(shape=bb.make_shape(2, 16, 128, bb.FMT_Q8_0, bb.QMODE_F16))),
    *(("scale must be finite", dict(shape=bb.Shape(2, 16, 128, 1, 272, 136, 0, x))) for x in (-0.1, float("nan"), float("inf"))),
    ("hd must be 128 or 256", dict(shape=bb.make_shape(2, 16, 64, bb.FMT_Q8_0))),
    ("fmt must be", dict(shape=bb.Shape(2, 16, 128, 3, 272, 136, 0, 0.1))),
    ("nkv and rows", dict(shape=bb.make_shape(0, 16, 128, bb.FMT_Q8_0))),
    ("too small", dict(shape=bb.make_shape(2, 16, 128, bb.FMT_Q8_0, rs=271))),
    ("fewer keys than n_nodes", dict(counts=(0, 3, 0))),
    ("fewer keys than n_nodes", dict(counts=())),
    ("null page", dict(k=None)),
    ("null page", dict(v=None)),
    ("null mask", dict(mask=None)),
    ("null mask", dict(Q=None)),
    ("null mask", dict(Oh=None)),
    ("null mask", dict(lse=None)),
    ("aligned", dict(mask=P + 4)),
    ("aligned", dict(Q=P + 2)),
    ("aligned", dict(Oh=P + 4)),
    ("aligned", dict(lse=P + 2)),
    ("2^24 rows", dict(shape=bb.make_shape(1, (1 << 24) + 4, 128, bb.FMT_Q8_0))),
    ("2^32 - 1 keys", dict(counts=(1 << 31, 1 << 31))),
    ("null workspace", dict()),
])
def test_tree_refuses(what, kw):
    refused(what, lambda: tree(**kw))


# ---------------------------------------------------------------- log probabilities
def logprobs(logits=P, type=bb.TYPE_F32, n_rows=3, vocab=1000, stride=1000, scale=1.0, given=P, n_given=2, n_top=5, logp=P, lse=P,
             entropy=P, top_id=P, top_logp=P):
    NoWorkspace().logprobs(logits, type, n_rows, vocab, stride, scale, given, n_given, n_top, logp, lse, entropy, top_id, top_logp)


@pytest.mark.parametrize("what,kw", [
    ("type must be", dict(type=3)),
    ("type must be", dict(type=-1)),
    ("n_rows must be", dict(n_rows=-1)),
    ("n_rows must be", dict(n_rows=(1 << 20) + 1)),
    ("vocab must be", dict(vocab=0)),
    ("vocab must be", dict(vocab=(1 << 24) + 1, stride=1 << 25)),
    ("row_stride must be", dict(stride=999)),
    ("row_stride must be", dict(stride=1 << 41)),
    ("scale must be", dict(scale=0.0)),
    ("scale must be", dict(scale=-1.0)),
    ("scale must be", dict(scale=float("nan"))),
    ("scale must be", dict(scale=float("inf"))),
    ("scale must be", dict(scale=1e-30)),
    ("scale must be", dict(scale=1e30)),
    ("n_given must be", dict(n_given=-1)),
    ("n_given must be", dict(n_given=1025)),
    ("n_given must be", dict(n_top=33)),
    ("n_given must be", dict(n_top=-1)),
    ("null argument", dict(logits=None)),
    ("null argument", dict(given=None)),
    ("null argument", dict(logp=None)),
    ("null argument", dict(top_id=None)),
    ("null argument", dict(top_logp=None)),
    ("aligned", dict(logits=P + 2)),
    ("aligned", dict(logits=P + 1, type=bb.TYPE_BF16)),
    ("aligned", dict(given=P + 2)),
    ("aligned", dict(lse=P + 1)),
    ("aligned", dict(entropy=P + 2)),
    ("null workspace", dict()),
    ("null workspace", dict(lse=None, entropy=None, n_given=0, given=None, logp=None, n_top=0, top_id=None, top_logp=None)),
])
def test_logprobs_refuses(what, kw):
    refused(what, lambda: logprobs(**kw))


def test_logprobs_no_rows_is_nothing():
    logprobs(n_rows=0, logits=None, given=None, logp=None, top_id=None, top_logp=None)


# ---------------------------------------------------------------- norm, rotation and append
def rope(**kw):
    f = dict(q_weight=P, k_weight=P, eps=1e-6, inv_freq=P, n_rot=128, type=bb.TYPE_F32)
    return bb.make_rope(**(f | kw))


def append(shape=None, counts=(64, 64), page_keys=64, pos0=60, rope_=None, Q=P, K=P, V=P, positions=P, n=4, q_out=P, k=P, v=P):
    shape = shape or bb.make_shape(2, 16, 128, bb.FMT_Q8_0)
    bb.append_rope(shape, pages(counts, k, v), page_keys, pos0, rope_ or rope(), Q, K, V, positions, n, q_out)


@pytest.mark.parametrize("what,kw", [
    ("hd must be 128 or 256", dict(shape=bb.make_shape(2, 16, 64, bb.FMT_Q8_0))),
    ("bad fmt or nkv", dict(shape=bb.make_shape(0, 16, 128, bb.FMT_Q8_0))),
    ("hb / rs too small", dict(shape=bb.make_shape(2, 16, 128, bb.FMT_Q8_0, rs=270))),
    ("page_keys", dict(page_keys=0)),
    ("past the last page", dict(pos0=125)),
    ("past the last page", dict(pos0=0xffffffff)),
    ("positions must be below 2^32", dict(counts=(64, 64, 64), page_keys=1 << 31, pos0=(1 << 32) - 2)),
    ("null page", dict(k=None)),
    ("null page", dict(v=None)),
    ("type must be", dict(rope_=rope(type=3))),
    ("n_rot must be", dict(rope_=rope(n_rot=130))),
    ("n_rot must be", dict(rope_=rope(n_rot=63))),
    ("null inv_freq", dict(rope_=rope(inv_freq=None))),
    ("eps must be", dict(rope_=rope(eps=-1.0))),
    ("eps must be", dict(rope_=rope(eps=float("nan")))),
    ("null K/V", dict(K=None)),
    ("null K/V", dict(V=None)),
    ("null K/V", dict(positions=None)),
    ("come together", dict(Q=None)),
    ("come together", dict(q_out=None)),
    ("multiple of n", dict(n=3)),
    ("multiple of n", dict(shape=bb.make_shape(2, 0, 128, bb.FMT_Q8_0))),
    ("strides must be at most", dict(rope_=rope(q_stride=1 << 33))),
    ("strides must be even", dict(rope_=rope(type=bb.TYPE_BF16, k_stride=257))),
    ("aligned", dict(Q=P + 2)),
    ("aligned", dict(K=P + 2)),
    ("aligned", dict(V=P + 1)),
    ("aligned", dict(q_out=P + 4)),
    ("aligned", dict(positions=P + 2)),
    ("aligned", dict(rope_=rope(q_weight=P + 2))),
    ("rs and hb must be multiples of 4", dict(shape=bb.make_shape(2, 16, 128, bb.FMT_F16, rs=514))),
    ("rs and hb must be multiples of 2", dict(shape=bb.make_shape(2, 16, 128, bb.FMT_Q8_0, rs=273))),
    ("is not 2-byte aligned", dict(k=P + 1)),
    ("is not 4-byte aligned", dict(shape=bb.make_shape(2, 16, 128, bb.FMT_F16), v=P + 2)),
])
def test_append_rope_refuses(what, kw):
    refused(what, lambda: append(**kw))


def test_append_rope_null_rope():
    s, t = bb.make_shape(2, 16, 128, bb.FMT_Q8_0), bb.PageTable(pages((64, 64)))
    rc = bb.lib().pa_hip_append_rope(C.byref(s), t.k, t.v, t.n, 64, 0, None, P, P, P, P, 4, P, None)
    assert rc == -1 and "null rope" in bb.last_error()


def test_append_rope_no_tokens_is_nothing():
    append(n=0, Q=None, K=None, V=None, positions=None, q_out=None)


# ---------------------------------------------------------------- row copies
PAGE_BYTES = 272 * 64


def layers(n, n_pages, base=P):
    """n layers of n_pages pages, all different."""
    at = [base + PAGE_BYTES * i for i in range(2 * n * n_pages)]
    return bb.LayerTable([bb.Pages(at[2 * n_pages * i:2 * n_pages * i + n_pages], at[2 * n_pages * i + n_pages:2 * n_pages * (i + 1)],
                                   [64] * n_pages, []) for i in range(n)])


A, B = layers(3, 2), layers(3, 2, base=P + 64 * PAGE_BYTES)
SHAPE = bb.make_shape(2, 1, 128, bb.FMT_Q8_0)


def with_page(table, i, value, tensor="k"):
    t = layers(table.layers, table.pages)
    t.k, t.v = type(table.k)(*table.k), type(table.v)(*table.v)
    getattr(t, tensor)[i] = value
    return t


@pytest.mark.parametrize("what,call", [
    ("bad shape", lambda: bb.copy_rows(bb.make_shape(2, 1, 128, bb.FMT_Q8_0, rs=271), A, B, 64, [0, 1], 0)),
    ("bad shape", lambda: bb.copy_rows(bb.make_shape(0, 1, 128, bb.FMT_Q8_0), A, B, 64, [0, 1], 0)),
    ("rs must be below", lambda: bb.copy_rows(bb.make_shape(2, 1, 128, bb.FMT_Q8_0, rs=1 << 26), A, B, 64, [0, 1], 0)),
    ("bad layer or page count", lambda: bb.copy_rows(SHAPE, A, B, 0, [0, 1], 0)),
    ("strictly increasing", lambda: bb.copy_rows(SHAPE, A, B, 64, [3, 3], 0)),
    ("strictly increasing", lambda: bb.copy_rows(SHAPE, A, B, 64, [3, 2], 0)),
    ("source positions past", lambda: bb.copy_rows(SHAPE, A, B, 64, [3, 128], 0)),
    ("source positions past", lambda: bb.copy_rows(SHAPE, A, B, 64, range(100, 130), 0)),
    ("destination positions past", lambda: bb.copy_rows(SHAPE, A, B, 64, [3, 5], 127)),
    ("destination positions past", lambda: bb.copy_rows(SHAPE, A, B, 64, [3, 5], 0xffffffff)),
    ("null destination page 1 of layer 2", lambda: bb.copy_rows(SHAPE, A, with_page(B, 5, None), 64, [3, 5], 63)),
    ("null source page 0 of layer 1", lambda: bb.copy_rows(SHAPE, with_page(A, 2, None, "v"), B, 64, [3, 5], 63)),
    ("a destination twice", lambda: bb.copy_rows(SHAPE, A, with_page(B, 2, B.k[0]), 64, [3, 5], 0)),
    ("a destination twice", lambda: bb.copy_rows(SHAPE, A, with_page(B, 0, B.v[0]), 64, [3, 5], 0)),
    ("at another place", lambda: bb.copy_rows(SHAPE, A, with_page(B, 2, A.k[0]), 64, [3, 5], 0)),
    ("at another place", lambda: bb.copy_rows(SHAPE, A, with_page(A, 1, A.k[0]), 64, [3, 5], 64)),
    ("at or behind their destination", lambda: bb.copy_rows(SHAPE, A, A, 64, [3, 5], 4)),
    ("at or behind their destination", lambda: bb.copy_rows(SHAPE, A, A, 64, range(0, 10), 1)),
    ("positions must be below 2^32", lambda: bb.copy_rows(SHAPE, A, layers(3, 3), 1 << 31, range(0, 4), (1 << 32) - 3)),
    ("positions must be below 2^32", lambda: bb.copy_rows(SHAPE, layers(3, 3), B, 1 << 31, range((1 << 32) - 5, (1 << 32) + 1), 0)),
    ("same number of layers", lambda: bb.copy_rows(SHAPE, A, layers(2, 2), 64, [0], 0)),
    ("same number of pages", lambda: bb.LayerTable([pages((64,)), pages((64, 64))])),
])
def test_copy_rows_refuses(what, call):
    refused(what, call)


def test_copy_rows_nothing_to_do():
    bb.copy_rows(SHAPE, A, B, 64, [], 0)
    bb.copy_rows(SHAPE, A, A, 64, [7, 8, 9], 7)                      # every row stays where it is: nothing is enqueued


def test_copy_rows_too_many_layers():
    assert bb.lib().pa_hip_copy_rows(C.byref(SHAPE), (1 << 20) + 1, A.k, A.v, 2, B.k, B.v, 2, 64, None, 0, 0, 5, None) == -1
    assert "bad layer" in bb.last_error()


def test_copy_rows_null_tables():
    z = C.POINTER(C.c_void_p)()
    for t in range(4):
        p = [A.k, A.v, B.k, B.v]
        p[t] = z
        assert bb.lib().pa_hip_copy_rows(C.byref(SHAPE), 3, p[0], p[1], 2, p[2], p[3], 2, 64, None, 0, 0, 5, None) == -1
        assert "null page table" in bb.last_error()
