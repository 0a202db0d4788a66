"""ptmi_batch_*: many requests through a model over one paged cache, against the model's own
token-by-token decode of each request alone (which the decode tests hold to the oracle).

Logits: 1e-5 of the largest, the bound of the decode step against the oracle (the orders of
the sums differ); with a bf16 cache every key and value is off by up to 2^-9 of itself.
"""
import numpy as np
import pytest

import pitorch_amd as pa
from pitorch_amd._ffi import PtmiError
from tests import _paged as R

pytestmark = pytest.mark.gpu

SMALL = (64, 160, 2, 4, 4, 512, 256)             # dim hidden layers heads kv_heads vocab seq_len
PADDED_HEAD = (108, 260, 2, 3, 3, 512, 160)      # head_dim 36
WIDE_HEAD = (256, 512, 2, 2, 2, 512, 96)         # head_dim 128
MIDDLE = (768, 1280, 2, 12, 12, 512, 640)        # head_dim 64; GEMMs that cut K


def alone(model, tokens, n_more):
    """Greedy tokens after `tokens`, and the logits after each position from the last given one on."""
    model.reset_kv()
    for t in tokens[:-1]:
        model.forward_step(int(t))
    out, logits, t = [], [], int(tokens[-1])
    for _ in range(n_more):
        t = model.forward_step(t)
        out.append(t)
        logits.append(model.logits())
    return out, logits


def close(got, want):
    assert np.max(np.abs(got - want)) <= 1e-5 * np.max(np.abs(want))


@pytest.mark.parametrize("cfg,page,lens", [
    (SMALL, 16, [1, 5, 16, 17, 70]), (SMALL, 7, [3, 130]), (PADDED_HEAD, 16, [40, 2, 33]), (WIDE_HEAD, 24, [30, 1]),
    (MIDDLE, 16, [200, 1, 65])])
def test_requests_together_as_alone(cfg, page, lens):
    """Prompts at once, then tokens together: each request's tokens and logits as if it were alone."""
    model = pa.Model(pa.synth_model(cfg, 5))
    prompts = [pa.seed_tokens(n + 40, n, cfg[5]).tolist() for n in lens]
    more = 6
    want = [alone(model, p, more) for p in prompts]
    n_pages = sum(R.pages_for(n + more, page) for n in lens)
    b = pa.Batch(model, len(lens) + 2, sum(lens), n_pages, page)
    model.close()                                            # the batch holds the weights
    new = {2 * i if i < 2 else i + 1: p for i, p in enumerate(prompts)}      # places 0, 2, 3, ..
    place = list(new)
    for k in range(more):
        got = b.step(new)
        for i, r in enumerate(place):
            assert got[r] == want[i][0][k], (k, i)
            close(b.logits(r), want[i][1][k])
            assert b.length(r) == lens[i] + k
        new = {r: [t] for r, t in got.items()}
    assert b.free_pages() >= 0
    b.close()


def test_requests_come_and_go():
    """Prompts in pieces beside single tokens, requests that end and whose pages others take, idle places."""
    cfg, page = SMALL, 8
    model = pa.Model(pa.synth_model(cfg, 6))
    rng = np.random.default_rng(2)
    want, prompts = {}, {}
    for i in range(12):
        prompts[i] = pa.seed_tokens(i + 9, int(rng.integers(1, 60)), cfg[5]).tolist()
        want[i] = alone(model, prompts[i], 10)
    b = pa.Batch(model, 4, 40, 4 * R.pages_for(70, page), page)
    total, place, todo, done = b.free_pages(), {}, list(range(12)), 0
    for _ in range(400):
        new, room = {}, 40
        for r in range(4):
            if r not in place and todo:
                place[r] = dict(req=todo.pop(0), fed=0, out=[])
            if r not in place:
                continue
            s = place[r]
            if len(s["out"]) == 10:
                assert s["out"] == want[s["req"]][0], s["req"]
                new[r] = None
                done += 1
                del place[r]
                continue
            p = prompts[s["req"]]
            n = min(len(p) - s["fed"], int(rng.integers(0, 14)), room) if s["fed"] < len(p) else min(1, room)
            if n:
                new[r] = p[s["fed"]:s["fed"] + n] if s["fed"] < len(p) else [s["out"][-1]]
                s["fed"] += n if s["fed"] < len(p) else 0
                room -= n
        got = b.step(new)
        for r, t in got.items():
            s = place[r]
            if s["fed"] == len(prompts[s["req"]]):
                close(b.logits(r), want[s["req"]][1][len(s["out"])])
                s["out"].append(t)
        if done == 12:
            break
    assert done == 12 and b.free_pages() == total
    assert all(b.length(r) == 0 for r in range(4))


def test_a_16_bit_cache():
    cfg = MIDDLE
    model = pa.Model(pa.synth_model(cfg, 7))
    p = pa.seed_tokens(3, 100, cfg[5]).tolist()
    _, logits = alone(model, p, 1)
    b = pa.Batch(model, 1, 100, 8, 16, pa.BF16)
    b.step({0: p})
    # scores and outputs are off by 2^-9 of their terms, at random: far under 1% of the logits
    err = np.linalg.norm(b.logits(0) - logits[0]) / np.linalg.norm(logits[0])
    assert 1e-7 < err < 1e-2


def test_sampled_tokens():
    """The tokens are those of the logits, each request by its own parameters and numbers."""
    model = pa.Model(pa.synth_model(SMALL, 8, 0.2))
    b = pa.Batch(model, 3, 64, 16)
    rng = np.random.default_rng(4)
    new = {0: [5, 9, 11], 2: [7]}
    args = dict(temperature=[0.7, 1.0, 1.3], top_k=[0, 0, 40], top_p=[0.9, 1.0, 1.0], min_p=[0.0, 0.0, 0.01])
    for _ in range(6):
        u = rng.random(3).astype(np.float32)
        got = b.step(new, u=u, **args)
        assert set(got) == {0, 2}
        for r in got:
            want, margin = R.sample(b.logits(r), float(np.float32(args["temperature"][r])), args["top_k"][r],
                                    float(np.float32(args["top_p"][r])), float(np.float32(args["min_p"][r])), float(u[r]))
            assert got[r] == want or margin < 512 * 2.0**-44
        new = {r: [t] for r, t in got.items()}
    greedy = b.step({1: [3]})[1]
    assert greedy == int(np.argmax(b.logits(1)))


def test_steps_that_do_not_fit_change_nothing():
    model = pa.Model(pa.synth_model(SMALL, 9))
    want = alone(model, [1, 2, 3, 4], 2)[0]
    b = pa.Batch(model, 2, 20, 3, 8)
    first = b.step({0: [1, 2, 3]})

    def refused(new, status=4):
        with pytest.raises(PtmiError) as e:
            b.step(new)
        assert e.value.status == status and b.length(0) == 3 and b.length(1) == 0 and b.free_pages() == 2
    refused({0: [4] * 11, 1: [4] * 10})                       # rows
    refused({0: [4], 1: [4] * 17})                            # pages
    refused({0: [512]}, 1)
    refused({0: [-1]}, 1)
    assert b.step({0: [4]})[0] == want[0] and first
    with pytest.raises(PtmiError):
        b.logits(1)
    big = pa.Batch(model, 1, 300, 64, 8)
    with pytest.raises(PtmiError) as e:
        big.step({0: [1] * 257})                              # seq_len
    assert e.value.status == 4
    assert big.step({}) == {} and big.length(0) == 0


def test_bad_batches():
    model = pa.Model(pa.synth_model(SMALL, 9))
    for args in ((0, 1, 1, 1), (8193, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0), (1, 1, 1 << 16, 1 << 15), (1, 1, 1, 1, 2)):
        with pytest.raises(PtmiError) as e:
            pa.Batch(model, *args)
        assert e.value.status == 1
    with pytest.raises(PtmiError) as e:
        pa.Batch(pa.Model(pa.synth_model((8, 8, 1, 1, 1, 262141, 4), 1)), 1, 1, 1)
    assert e.value.status == 1
    b = pa.Batch(model, 2, 4, 4)
    for request in (-1, 2):
        with pytest.raises(ValueError):
            b.step({request: [1]})
    assert b.free_pages() == 4


def test_the_blob_is_not_read_again():
    """A batch takes the model's weights as they are on the GPU: the host's may be gone, and the model too."""
    blob = pa.synth_model(SMALL, 9)
    model = pa.Model(blob)
    want = alone(model, [1, 2, 3], 2)[0]
    blob[:] = 0
    b = pa.Batch(model, 1, 8, 8)
    model.close()
    t = b.step({0: [1, 2, 3]})[0]
    assert [t, b.step({0: [t]})[0]] == want


def test_the_longest_request():
    """All of seq_len, the last position included."""
    cfg = WIDE_HEAD
    model = pa.Model(pa.synth_model(cfg, 10))
    p = pa.seed_tokens(5, cfg[6] - 1, cfg[5]).tolist()
    want, logits = alone(model, p, 2)
    b = pa.Batch(model, 1, 96, 3, 32)
    t = b.step({0: p})[0]
    assert t == want[0]
    assert b.step({0: [t]})[0] == want[1]
    close(b.logits(0), logits[1])
    with pytest.raises(PtmiError):
        b.step({0: [1]})
