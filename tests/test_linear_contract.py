"""dispatch_layout of conv_causal, attn_linear and sample_logits: sizes,
threads and refusals."""
import pytest

import qmr
from linear_cases import f32_word

CONV = dict(seqs=3, tokens=10, channels=30, width=4, xs=33, ys=30, silu=1, bias=1, pool=5, keep=1)
LINEAR = dict(seqs=3, tokens=10, hk=2, hv=6, dk=32, dv=64, qs=512, ks=512, vs=512, sa=6, sb=8, sz=384, so=390, most=7,
              gates=1, delta=1, scale=f32_word(0.2), qk=f32_word(1e-6), out=f32_word(1e-6), pool=5, keep=1)
SAMPLE = dict(rows=4, vocab=1000, stride=1003)
BASE = {"conv_causal": CONV, "attn_linear": LINEAR, "sample_logits": SAMPLE}


def layout(name, **change):
    return qmr.dispatch_layout(name, list({**BASE[name], **change}.values()))


def test_sizes():
    assert layout("conv_causal") == ([4 * (9 * 33 + 30), 480, 120, 16, 12, 5 * 3 * 30 * 4, 1200], 10 * 8)
    assert layout("conv_causal", bias=0, width=2)[0] == [4 * (9 * 33 + 30), 240, 0, 16, 12, 600, 1200]
    qk, vz = 4 * (9 * 512 + 64), 4 * (9 * 384 + 384)
    assert layout("attn_linear") == (
        [qk, qk, 4 * (9 * 512 + 384), 240, 4 * (9 * 8 + 6), 24, 24, vz, 256, 16, 12, 5 * 6 * 32 * 64 * 4,
         4 * (9 * 390 + 384)], 10 * 6 * 32)
    sizes, _ = layout("attn_linear", gates=0, delta=0, out=0, sa=0, sb=0, sz=0)
    assert sizes[3:9] == [24, 0, 0, 0, 0, 0]
    assert layout("sample_logits") == ([4 * (3 * 1003 + 1000)] + [16] * 7, 4096)
    # Pools past 2^32 floats.
    assert layout("attn_linear", pool=1 << 20)[0][11] == (1 << 20) * 6 * 32 * 64 * 4


NAN, INF = f32_word(float("nan")), f32_word(float("inf"))


@pytest.mark.parametrize("change,match", [
    (dict(seqs=0), "nonzero"), (dict(tokens=0), "nonzero"), (dict(channels=0), "nonzero"), (dict(pool=0), "nonzero"),
    (dict(width=1), "taps"), (dict(width=5), "taps"), (dict(xs=29), "stride"), (dict(ys=29), "stride"),
    (dict(silu=2), "switches"), (dict(bias=2), "switches"), (dict(keep=2), "switches"), (dict(pool=1 << 31), "slots"),
    (dict(channels=1 << 23, xs=1 << 23, ys=1 << 23), "channels"),
    (dict(tokens=1 << 31, channels=64, xs=64, ys=64), "overflow"), (dict(seqs=1 << 27), "overflow")])
def test_conv_refusals(change, match):
    with pytest.raises(qmr.QmrError, match=match):
        layout("conv_causal", **change)


@pytest.mark.parametrize("change,match", [
    (dict(seqs=0), "nonzero"), (dict(tokens=0), "nonzero"), (dict(hk=0), "nonzero"), (dict(dk=0), "nonzero"),
    (dict(most=0), "nonzero"), (dict(pool=0), "nonzero"), (dict(hv=5), "multiple of the key heads"),
    (dict(dk=36), "multiples of 8"), (dict(dv=264, vs=2000, sz=2000, so=2000), "at most 256"), (dict(qs=63), "stride"),
    (dict(ks=63), "stride"), (dict(vs=383), "stride"), (dict(sa=5), "stride"), (dict(sb=5), "stride"),
    (dict(sb=0), "stride"), (dict(sz=383), "stride"), (dict(so=383), "stride"), (dict(gates=2), "switches"),
    (dict(delta=2), "switches"), (dict(keep=2), "switches"), (dict(scale=0), "scale"), (dict(scale=NAN), "scale"),
    (dict(scale=INF), "scale"), (dict(qk=NAN), "epsilons"), (dict(qk=0x80000000), "epsilons"), (dict(out=INF), "epsilons"),
    (dict(out=f32_word(-1.0)), "epsilons"), (dict(pool=1 << 31), "slots"), (dict(seqs=1 << 20), "overflow"),
    (dict(tokens=1 << 26), "overflow"), (dict(seqs=1 << 19), "overflow"),
    (dict(hk=1, hv=65536, dk=8, dv=8, qs=8, ks=8, vs=1 << 19, sa=65536, sb=65536, sz=1 << 19, so=1 << 19), "too many heads")])
def test_linear_refusals(change, match):
    with pytest.raises(qmr.QmrError, match=match):
        layout("attn_linear", **change)


@pytest.mark.parametrize("change,match", [
    (dict(rows=0), "nonzero"), (dict(vocab=0), "nonzero"), (dict(stride=999), "stride"), (dict(rows=1 << 22), "overflow"),
    (dict(vocab=(1 << 24) + 1, stride=1 << 25), "at most 2\\^24")])
def test_sample_refusals(change, match):
    with pytest.raises(qmr.QmrError, match=match):
        layout("sample_logits", **change)


@pytest.mark.parametrize("name", list(BASE))
def test_parameter_counts(name):
    words = list(BASE[name].values())
    for wrong in (words[:-1], [*words, 0]):
        with pytest.raises(qmr.QmrError, match=f"expected {len(words)} parameters"):
            qmr.dispatch_layout(name, wrong)
