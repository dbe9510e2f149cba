"""``rope_tables`` against its formulas and the models that scale their angles (CPU)."""
import math

import pytest
import torch


def angles(n, freq):
    return torch.arange(n, dtype=torch.float64)[:, None] * torch.tensor(freq, dtype=torch.float64)


def check(tables, n, freq, gain=1.0):
    """fp32 of the 64-bit values: half a step, 2^-24 of the gain, and 2^-40 for the
    angles' own rounding (positions below 2^12)."""
    for got, want in zip(tables, (angles(n, freq).cos(), angles(n, freq).sin())):
        assert got.dtype == torch.float32
        assert ((got.double() - want * gain).abs() <= gain * (2.0 ** -24 + 2.0 ** -40)).all()


@pytest.mark.parametrize("rot,theta", [(128, 1e6), (32, 1e4), (2, 10.0)])
def test_plain_and_linear(rot, theta):
    from d2sd_b200 import rope_tables
    freq = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    check(rope_tables(300, rot, theta, "cpu"), 300, freq)
    check(rope_tables(300, rot, theta, "cpu", scaling={"type": "linear", "factor": 4}), 300,
          [x / 4 for x in freq])


@pytest.mark.parametrize("truncate", [None, True, False])
@pytest.mark.parametrize("rot,theta,f,L,fast,slow", [(64, 150000.0, 32.0, 4096, 32, 1), (128, 1e6, 4.0, 32768, 32, 1),
                                                     (64, 1e4, 8.0, 2048, 16, 2), (128, 1e4, 1.0, 4096, 32, 1)])
def test_yarn(rot, theta, f, L, fast, slow, truncate):
    from d2sd_b200 import rope_tables
    s = {"type": "yarn", "factor": f, "original": L, "beta_fast": fast, "beta_slow": slow}
    if truncate is not None:
        s["truncate"] = truncate
    # column c's wave turns L * theta^(-2 c / rot) / (2 pi) times over L positions
    lo, hi = (rot / 2 * math.log(L / (2 * math.pi * t)) / math.log(theta) for t in (fast, slow))
    if truncate is not False:
        lo, hi = math.floor(lo), math.ceil(hi)
    lo, hi = max(lo, 0), min(hi, rot - 1)
    freq = []
    for c in range(rot // 2):
        ramp = min(max((c - lo) / (hi - lo), 0.0), 1.0)
        x = theta ** (-2 * c / rot)
        freq.append(x * (1 - ramp) + x / f * ramp)
    check(rope_tables(4000, rot, theta, "cpu", scaling=s), 4000, freq, 0.1 * math.log(f) + 1 if f > 1 else 1.0)


def test_the_angles_of_gpt_oss():
    """The configuration's own scaling (its defaults: YaRN without truncation) gives the
    model's frequencies and gain, to the fp32 of the model's own table."""
    transformers = pytest.importorskip("transformers")
    from d2sd_b200 import rope_tables
    config = transformers.GptOssConfig()
    from transformers.models.gpt_oss.modeling_gpt_oss import GptOssRotaryEmbedding
    rotary = GptOssRotaryEmbedding(config)
    p = config.rope_parameters
    assert p["rope_type"] == "yarn" and p["truncate"] is False
    scaling = {"type": "yarn", "factor": p["factor"], "original": p["original_max_position_embeddings"],
               "beta_fast": p["beta_fast"], "beta_slow": p["beta_slow"], "truncate": p["truncate"]}
    D = config.head_dim
    cos, sin = rope_tables(2, D, p["rope_theta"], "cpu", scaling=scaling)
    gain = (cos[0].double() ** 2 + sin[0].double() ** 2).sqrt()
    assert ((gain - rotary.attention_scaling).abs() <= 1e-6).all()
    # the angle of position 1 is the frequency
    freq = torch.atan2(sin[1].double(), cos[1].double())
    assert ((freq / rotary.inv_freq.double() - 1).abs() <= 2.0 ** -20).all()


def test_refusals():
    from d2sd_b200 import rope_tables
    yarn = {"type": "yarn", "factor": 4.0, "original": 4096}
    for err, kw in [(ValueError, dict(scaling=dict(yarn, attention_factor=1.0))),
                    (ValueError, dict(scaling=dict(yarn, mscale=1.0))),
                    (ValueError, dict(scaling={"type": "linear", "factor": 2.0, "truncate": False})),
                    (NotImplementedError, dict(scaling={"type": "dynamic", "factor": 2.0})),
                    (NotImplementedError, dict(scaling={"factor": 2.0})),
                    (KeyError, dict(scaling={"type": "yarn", "factor": 2.0}))]:
        with pytest.raises(err):
            rope_tables(8, 64, 1e4, "cpu", **kw)
    for n, rot in ((0, 64), (8, 0), (8, 63)):
        with pytest.raises(ValueError):
            rope_tables(n, rot, 1e4, "cpu")
