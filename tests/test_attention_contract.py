"""dispatch_layout of the attention names: sizes, threads and refusals."""
import pytest

import qmr
from attention_cases import f32_word

ROPE = dict(tokens=7, heads=3, dim=64, rotary=32, xs=192, ys=200, adjacent=0, dealt=0, axes=2, n0=10, n1=6, n2=0, n3=0)
APPEND = dict(seqs=2, tokens=5, heads=6, kv=2, dim=64, rotary=64, qs=640, ks=640, vs=640, os=384, adjacent=0, dealt=1,
              axes=3, n0=12, n1=10, n2=10, n3=0, eps=f32_word(1e-6), page=64, pages=9, columns=4)
ATTEND = dict(seqs=2, tokens=5, heads=6, kv=2, dim=64, qs=384, os=400, page=64, pages=9, columns=4, keys=200, causal=1,
              window=0, scale=f32_word(0.125))


def layout(name, base, **change):
    return qmr.dispatch_layout(name, list({**base, **change}.values()))


def test_sizes():
    assert layout("rope_axes", ROPE) == ([4 * (6 * 192 + 192), 4 * 2 * 7, 64, 4 * (6 * 200 + 192)], 7 * 3 * 32)
    cache = 9 * 2 * 64 * 64 * 2
    q, k = 4 * (4 * 640 + 384), 4 * (4 * 640 + 128)
    for kind in ("bf16", "f16"):
        assert layout("kv_append_rope_" + kind, APPEND) == (
            [q, k, k, 256, 256, 4 * 3 * 5, 128, 12, 8, 32, cache, cache, 4 * 5 * 384], 5 * 10 * 32)
        assert layout("attn_paged_" + kind, ATTEND) == (
            [4 * 5 * 384, 12, 8, 32, cache, cache, 4 * (4 * 400 + 384)], 5 * 6 * 32)
    sizes, _ = layout("kv_append_rope_f16", APPEND, eps=0, heads=0, qs=0, os=0, rotary=0, axes=0, n0=0, n1=0, n2=0, dealt=0)
    assert sizes[0] == sizes[3] == sizes[4] == sizes[5] == sizes[6] == sizes[12] == 0
    # A pool past 2^32 halves.
    sizes, _ = layout("attn_paged_f16", ATTEND, pages=1 << 21)
    assert sizes[4] == (1 << 21) * 2 * 64 * 64 * 2


@pytest.mark.parametrize("change,match", [
    (dict(tokens=0), "nonzero"), (dict(heads=0, xs=0), "nonzero"), (dict(rotary=0, n0=0, n1=0), "nonzero"),
    (dict(rotary=31), "even part"), (dict(rotary=66, n0=17, n1=16), "even part"), (dict(xs=191), "stride"),
    (dict(ys=191), "stride"), (dict(axes=0), "one through four"), (dict(axes=5), "one through four"),
    (dict(axes=1), "no axis"), (dict(n0=11), "add up"), (dict(adjacent=2), "0 or 1"), (dict(dealt=2), "0 or 1"),
    (dict(dealt=1, n0=7, n1=9), "dealt"), (dict(dim=258, xs=774, ys=774), "at most 256"),
    (dict(dim=63, xs=192), "even"), (dict(tokens=1 << 31), "overflow")])
def test_rope_refusals(change, match):
    with pytest.raises(qmr.QmrError, match=match):
        layout("rope_axes", ROPE, **change)


@pytest.mark.parametrize("change,match", [
    (dict(seqs=0), "nonzero"), (dict(kv=0), "nonzero"), (dict(pages=0), "nonzero"), (dict(dim=60), "multiples of 8"),
    (dict(dim=264), "256"), (dict(heads=7), "multiple of the key-value heads"), (dict(page=48), "power of two"),
    (dict(page=16), "power of two"), (dict(eps=f32_word(-1.0)), "epsilon"), (dict(eps=f32_word(float("nan"))), "epsilon"),
    (dict(eps=f32_word(float("inf"))), "epsilon"), (dict(eps=0x80000000), "epsilon"), (dict(qs=383), "stride"),
    (dict(ks=127), "stride"), (dict(vs=127), "stride"), (dict(os=383), "stride"),
    (dict(columns=1 << 26), "too many positions"), (dict(rotary=0, n0=0, n1=0, n2=0), "axes")])
def test_append_refusals(change, match):
    with pytest.raises(qmr.QmrError, match=match):
        layout("kv_append_rope_bf16", APPEND, **change)


@pytest.mark.parametrize("change,match", [
    (dict(seqs=0), "nonzero"), (dict(heads=0), "nonzero"), (dict(columns=0), "nonzero"), (dict(heads=5), "multiple"),
    (dict(keys=0), "most keys"), (dict(keys=257), "most keys"), (dict(causal=2), "causal"),
    (dict(causal=0, window=4), "window"), (dict(window=1 << 31), "window"), (dict(scale=f32_word(0.0)), "scale"),
    (dict(scale=f32_word(float("inf"))), "scale"), (dict(scale=f32_word(-1.0)), "scale"), (dict(qs=380), "stride"),
    (dict(os=383), "stride"), (dict(page=96), "power of two"), (dict(pages=0), "nonzero")])
def test_attend_refusals(change, match):
    with pytest.raises(qmr.QmrError, match=match):
        layout("attn_paged_f16", ATTEND, **change)


@pytest.mark.parametrize("name,base", [("rope_axes", ROPE), ("kv_append_rope_f16", APPEND), ("attn_paged_bf16", ATTEND)])
def test_parameter_counts(name, base):
    for words in (list(base.values())[:-1], [*base.values(), 0]):
        with pytest.raises(qmr.QmrError, match="parameters"):
            qmr.dispatch_layout(name, words)
    with pytest.raises(qmr.QmrError, match="Unknown GPU kernel"):
        qmr.dispatch_layout(name + "_f32", list(base.values()))
