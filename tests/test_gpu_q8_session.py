"""Inference sessions with 8-bit activations (bmx_model_set_act_quant): prefill, token-by-token decode and batched greedy loops against the same
walk in 64 bits, which rounds where the session rounds (codes of weights and operands, gate | up and the branches in bf16).

Bound: a code whose quotient lies within the kernels' error of a tie may fall on the other side (about one code in ten thousand in a norm, one
in a hundred behind the bf16 roundings), which moves its value by a step, 1/127 of its row's largest. Behind one half of a layer that is 1 to
2 % of the branch (tests/test_gpu_q8_ops.py), independent between the four to six halves of these models: sqrt(6) * 2 % = 5 % of the
logits' 2-norm."""
import ctypes as C
import os

import numpy as np
import pytest

import bmapi
from bmcapi import bf16_round

pytestmark = pytest.mark.gpu
F32, BF16 = bmapi.BM_PRECISION_FP32, bmapi.BM_PRECISION_BF16
FAR = 0.05


class Walk:
    """The session's arithmetic in float64 over whole sequences."""

    def __init__(self, a, w, precision):
        self.a, self.w = a, w
        to8 = self.to8
        L = a.n_layers
        self.qkv = [to8(np.concatenate([w["qw"][l], w["kw"][l], w["vw"][l]])) for l in range(L)]
        self.o, self.down = [to8(w["ow"][l]) for l in range(L)], [to8(w["down"][l]) for l in range(L)]
        self.gu = [to8(np.concatenate([w["gate"][l], w["up"][l]])) for l in range(L)]
        self.head = (bf16_round(w["embed"]) if precision == BF16 else w["embed"]).astype(np.float64)

    @staticmethod
    def to8(v):
        v = np.asarray(v, np.float64)
        s = np.abs(v).max(1, keepdims=True) / 127
        return np.rint(v / s) * s

    @staticmethod
    def rms(x, w):
        return x / np.sqrt(np.mean(x * x, axis=1, keepdims=True) + 1e-5) * w

    @staticmethod
    def attention(q, k, v):
        T = len(q)
        s = np.einsum("qhd,khd->hqk", q, k) / np.sqrt(q.shape[-1])
        s = np.where(np.tril(np.ones((T, T), bool)), s, -np.inf)
        p = np.exp(s - s.max(-1, keepdims=True))
        return np.einsum("hqk,khd->qhd", p / p.sum(-1, keepdims=True), v).reshape(T, -1)

    def logits(self, tokens, bf16_cache_from=None):
        """[T, V] for one sequence. From row bf16_cache_from on, keys and values are read from a bf16 cache (a prompt's own rows are not)."""
        a, w, T = self.a, self.w, len(tokens)
        HD, NH, NKV, H = a.head_dim, a.n_heads, a.n_kv_heads, a.hidden_dim
        half = lambda v: bf16_round(v.astype(np.float32)).astype(np.float64)
        ang = np.arange(T)[:, None] * (1.0 / a.rope_theta ** (np.arange(0, HD, 2) / HD))
        cos, sin = np.cos(ang)[:, None], np.sin(ang)[:, None]
        rot = lambda v: np.concatenate([v[..., :HD // 2] * cos - v[..., HD // 2:] * sin, v[..., :HD // 2] * sin + v[..., HD // 2:] * cos], -1)
        x = w["embed"][np.asarray(tokens)].astype(np.float64)
        for l in range(a.n_layers):
            qkv = self.to8(self.rms(x, w["ln1w"][l])) @ self.qkv[l].T
            q, k, v = np.split(qkv, [NH * HD, (NH + NKV) * HD], axis=1)
            q, k, v = rot(q.reshape(T, NH, HD)), rot(k.reshape(T, NKV, HD)), v.reshape(T, NKV, HD)
            k, v = np.repeat(k, NH // NKV, 1), np.repeat(v, NH // NKV, 1)
            att = self.attention(q, k, v)
            if bf16_cache_from is not None:
                att[bf16_cache_from:] = self.attention(q, half(k), half(v))[bf16_cache_from:]
            x = x + half(self.to8(att) @ self.o[l].T)
            gu = half(self.to8(self.rms(x, w["ln2w"][l])) @ self.gu[l].T)
            g, u = gu[:, :H], gu[:, H:]
            branch = self.to8(g / (1 + np.exp(-g)) * u) @ self.down[l].T
            x = x + (branch if l == a.n_layers - 1 else half(branch))
        return self.rms(x, w["lnfw"]) @ self.head.T


class Session:
    def __init__(self, lib, name, precision, NB=1, MS=64, act=8, quant=0, seed=3, kv_bf16=0):
        self.lib, self.NB = lib, NB
        self.a = bmapi.make_arch(name)
        self.a.precision = precision
        self.w = bmapi.make_weights(self.a, seed=seed, layer_scale=8.0)
        rng = np.random.default_rng(seed)
        for k in ("ln1w", "ln2w", "lnfw"):
            self.w[k] = (1 + 0.1 * rng.standard_normal(self.w[k].shape)).astype(np.float32)
        path = f"/tmp/bm_q8s_{os.getpid()}.bin"
        bmapi.write_bin_checkpoint(path, self.a, self.w)
        self.ctx = lib.bm_create(bmapi.BM_DEVICE_CUDA)
        self.model = lib.bm_create_model(self.ctx, C.byref(self.a))
        lib.bm_load_weights(self.model, path.encode())
        os.unlink(path)
        assert lib.bmx_model_set_act_quant(self.model, act) == 0 and lib.bmx_model_set_quant(self.model, quant) == 0
        self.sess = lib.bmx_create_session_kv(self.ctx, self.model, NB, MS, kv_bf16)

    def vec(self, p):
        assert p
        return np.ctypeslib.as_array(p, shape=(self.NB, self.a.vocab_size)).copy()

    def forward(self, tokens):
        t = np.ascontiguousarray(tokens, np.int32)
        return self.vec(self.lib.bm_forward(self.sess, bmapi.as_int_ptr(t), len(t)))[0]

    def close(self):
        if self.sess:
            self.lib.bm_destroy_session(self.sess)
        self.lib.bm_destroy_model(self.model)
        self.lib.bm_destroy(self.ctx)


def near(got, ref):
    return np.linalg.norm(got - ref) <= FAR * np.linalg.norm(ref)


@pytest.mark.parametrize("name,precision", [("tiny", F32), ("tiny", BF16), ("small", BF16), ("gqa", F32), ("gqa", BF16)])
def test_steps_and_prefill(product, name, precision):
    s = Session(product, name, precision)
    ref = Walk(s.a, s.w, precision)
    toks = bmapi.lcg_tokens(24, s.a.vocab_size, seed=9)
    want = ref.logits(toks)
    for i in range(12):   # the third step on replays a graph
        assert near(s.vec(s.lib.bm_step(s.sess, int(toks[i])))[0], want[i]), i
    s.lib.bm_reset_session(s.sess)
    assert near(s.forward(toks[:17]), want[16])
    for i in range(17, 24):
        assert near(s.vec(s.lib.bm_step(s.sess, int(toks[i])))[0], want[i]), i
    # a longer prompt after a shorter one: the prefill buffers grow
    s.lib.bm_reset_session(s.sess)
    assert near(s.forward(toks), want[23])
    s.close()


@pytest.mark.parametrize("NB,n_prompt", [(2, 5), (3, 12), (8, 9), (40, 16), (130, 8)])
def test_batched_greedy(product, NB, n_prompt):
    """Every sequence of a batch against its own walk over the prompt and the tokens that the session chose. A chosen token has to be the walk's
    largest logit up to the bound on both."""
    n_new = 6
    s = Session(product, "gqa", BF16, NB=NB, MS=40)
    ref = Walk(s.a, s.w, BF16)
    V = s.a.vocab_size
    prompt = bmapi.lcg_tokens(NB * n_prompt, V, seed=NB).reshape(NB, n_prompt)
    out = np.zeros((NB, n_new), np.int32)
    assert s.lib.bmx_session_generate_greedy(s.sess, bmapi.as_int_ptr(np.ascontiguousarray(prompt)), n_prompt, n_new, bmapi.as_int_ptr(out)) == 0
    last = s.vec(s.lib.bmx_session_logits(s.sess))
    for b in list(range(min(NB, 6))) + [NB - 1]:
        want = ref.logits(np.concatenate([prompt[b], out[b][:-1]]))[n_prompt - 1:]
        assert near(last[b], want[-1]), b
        for i in range(n_new):
            assert want[i].max() - want[i][out[b, i]] <= 2 * FAR * np.linalg.norm(want[i]) / np.sqrt(V) * 5, (b, i)   # one logit: five times the mean error
    s.close()


@pytest.mark.parametrize("kv_bf16,variables", [(1, ()), (0, ("BM_NO_TC_DECODE",)), (0, ("BM_NO_GRAPH", "BM_NO_PDL"))])
def test_other_session_settings(product, monkeypatch, kv_bf16, variables):
    """A bf16 KV cache, no split-bf16 classifier (and so no prefill in one pass), no graph."""
    for v in variables:
        monkeypatch.setenv(v, "1")
    s = Session(product, "gqa", BF16, NB=9, MS=32, kv_bf16=kv_bf16)
    ref = Walk(s.a, s.w, BF16)
    prompt = bmapi.lcg_tokens(9 * 10, s.a.vocab_size, seed=2).reshape(9, 10)
    out = np.zeros((9, 4), np.int32)
    assert s.lib.bmx_session_generate_greedy(s.sess, bmapi.as_int_ptr(np.ascontiguousarray(prompt)), 10, 4, bmapi.as_int_ptr(out)) == 0
    last = s.vec(s.lib.bmx_session_logits(s.sess))
    for b in range(9):
        assert near(last[b], ref.logits(np.concatenate([prompt[b], out[b][:-1]]), 10 if kv_bf16 else None)[-1]), b
    s.close()


def test_bytes_and_refusals(product):
    s = Session(product, "gqa", BF16, NB=8)
    a = s.a
    QD, KV = a.n_heads * a.head_dim, a.n_kv_heads * a.head_dim
    rows = (QD + 2 * KV, a.dim), (a.dim, QD), (2 * a.hidden_dim, a.dim), (a.dim, a.hidden_dim)
    layer = sum(oc * c + 4 * oc for oc, c in rows)
    assert product.bmx_session_algorithmic_weight_bytes(s.sess) == a.n_layers * layer + a.vocab_size * a.dim * 2
    assert product.bmx_session_weight_bytes(s.sess) == a.n_layers * layer + a.vocab_size * a.dim * 2 * 2   # the head as [w | w]
    s.close()
    both = Session(product, "tiny", F32, quant=8)
    assert not both.sess
    both.close()


def test_other_sessions_of_the_model_stay_as_they_are(product):
    """A session made before the switch, and one after it is off again, give the bits of a plain model's session."""
    toks = bmapi.lcg_tokens(11, 512, seed=4)
    plain = Session(product, "tiny", F32, act=0)
    want = [plain.vec(product.bm_step(plain.sess, int(t)))[0] for t in toks]
    assert product.bmx_model_set_act_quant(plain.model, 8) == 0
    eight = product.bm_create_session(plain.ctx, plain.model)
    assert product.bmx_model_set_act_quant(plain.model, 0) == 0
    again = product.bm_create_session(plain.ctx, plain.model)
    product.bm_reset_session(plain.sess)
    for i, t in enumerate(toks):
        x, y = (plain.vec(product.bm_step(h, int(t)))[0] for h in (again, eight))
        assert np.array_equal(x, want[i]) and not np.array_equal(y, want[i])
    product.bm_destroy_session(eight)
    product.bm_destroy_session(again)
    plain.close()
