"""Token by token decoding of a small recurrent (state space) model: the projections are matvecs, and the
norm, the short convolution, the selective scan and the draw are the operators of sequence models.
One step is recorded once; every token submits it again, its states brought up to date in place.
The weights are random; the check runs the same model in NumPy.

    python examples/state_space_decode.py [tokens] [width] [vocabulary]
"""
import sys

import numpy as np

import charmnumeric_b200 as cnp

TOKENS = int(sys.argv[1]) if len(sys.argv) > 1 else 24
WIDTH = int(sys.argv[2]) if len(sys.argv) > 2 else 64
VOCABULARY = int(sys.argv[3]) if len(sys.argv) > 3 else 1000
INNER, STATES, TAPS, TEMPERATURE, TOP_K = 2 * WIDTH, 16, 4, 0.8, 40

rng = np.random.default_rng(1)
embedding = rng.standard_normal((VOCABULARY, WIDTH))
par = {"norm": 1 + 0.1 * rng.standard_normal(WIDTH), "in": rng.standard_normal((2 * INNER, WIDTH)) / WIDTH ** 0.5,
       "taps": rng.standard_normal((INNER, TAPS)) / TAPS ** 0.5, "delta": rng.standard_normal((INNER, INNER)) * 0.1 / INNER ** 0.5,
       "bc": rng.standard_normal((2 * STATES, INNER)) / INNER ** 0.5, "A": -np.tile(np.arange(1.0, STATES + 1), (INNER, 1)),
       "D": np.ones(INNER), "bias": np.full(INNER, -3.0), "out": rng.standard_normal((WIDTH, INNER)) / INNER ** 0.5}
numbers = rng.random(TOKENS)

interface = cnp.CharmNumericInterface(device=0)
p = {k: cnp.asarray(v) for k, v in par.items()}
head = cnp.asarray(embedding)
token_in, u = cnp.zeros((WIDTH,)), cnp.zeros((1,))
inputs, state = cnp.zeros((1, TAPS - 1, INNER)), cnp.zeros((1, INNER, STATES))


def as_sequence(v):
    out = cnp.zeros((1, 1, v.shape[0]))
    out[0, 0, :] = v
    return out


def as_vector(v):
    out = cnp.zeros((v.shape[2],))
    out[...] = v[0, 0, :]
    return out


def step():
    h = cnp.rms_norm(token_in, p["norm"])
    xz = p["in"] @ h
    x, _ = cnp.causal_conv(as_sequence(xz[:INNER]), p["taps"], state=inputs, activation="silu", inplace=True)
    flat = as_vector(x)
    bc = p["bc"] @ flat
    y, _ = cnp.selective_scan(x, as_sequence(p["delta"] @ flat), p["A"], as_sequence(bc[:STATES]), as_sequence(bc[STATES:]),
                              D=p["D"], z=as_sequence(xz[INNER:]), delta_bias=p["bias"], state=state, inplace=True)
    last, _ = cnp.rms_norm(p["out"] @ as_vector(y), p["norm"], residual=token_in)
    return cnp.random.sample(head @ last, u, temperature=TEMPERATURE, top_k=TOP_K)


recorded = cnp.record(step)
token, tokens, logp = 0, [], []
for i in range(TOKENS):
    token_in[...] = embedding[token]
    u[...] = float(numbers[i])
    token_array, logp_array = recorded.run(interface)
    token = int(token_array.get(interface)[0])
    tokens.append(token)
    logp.append(float(logp_array.get(interface)[0]))
print("tokens:", tokens)


def norm(v):
    return v / np.sqrt((v * v).mean() + 1e-6) * par["norm"]


past, h, token = np.zeros((TAPS - 1, INNER)), np.zeros((INNER, STATES)), 0
for i in range(TOKENS):
    e = embedding[token]
    xz = par["in"] @ norm(e)
    window = np.vstack([past, xz[:INNER]])
    past = window[1:]
    s = (window.T * par["taps"]).sum(1)
    x = s / (1 + np.exp(-s))
    bc, dt = par["bc"] @ x, np.logaddexp(0.0, par["delta"] @ x + par["bias"])
    h = np.exp(dt[:, None] * par["A"]) * h + (dt * x)[:, None] * bc[:STATES]
    z = xz[INNER:]
    y = (h @ bc[STATES:] + par["D"] * x) * z / (1 + np.exp(-z))
    logits = embedding @ norm(par["out"] @ y + e)
    best = np.sort(np.argsort(-logits, kind="stable")[:TOP_K])
    w = np.exp((logits[best] - logits.max()) / TEMPERATURE)
    at = int(np.searchsorted(np.cumsum(w), numbers[i] * w.sum(), side="right"))
    token = int(best[at])
    assert token == tokens[i], (i, token, tokens[i])
    assert abs(np.log(w[at] / w.sum()) - logp[i]) < 1e-8
print("Match: True")
