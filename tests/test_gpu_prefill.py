"""A client's prompt from its own pass in the clear into the encrypted decoder: the K and V rows of prefill.prefill loaded
into model.Decoder's caches (two layers at N = 2^14, the chain of tests/test_gpu_model.py), the next token decoded under
encryption, against the 64-bit model of the whole sequence."""
import numpy as np
import pytest
import torch

from perseus_b200 import bootstrap as BS
from perseus_b200 import fhe
from perseus_b200 import linear as LIN
from perseus_b200 import model as M
from perseus_b200 import prefill as PF

pytestmark = pytest.mark.gpu


def test_prefilled_caches_decode_on():
    logn = 14
    cfg = M.ModelCfg(layers=2, d=192, width=256, heads=3, head_dim=64, mlp=768, tokens=64, radix_bits=3)
    prm = BS.Params(1 << logn, K=24, r=3, per_group=5)
    ch = fhe.Chain(logn, tuple(fhe.ntt_primes(50, logn, 27)), tuple(fhe.ntt_primes(50, logn, 10, skip=27)), 3)
    lay = M.B.layout(ch.n // 2, cfg.width, cfg.heads, cfg.head_dim, cfg.tokens, cfg.radix_bits)
    steps = sorted(set(BS.rot_steps(prm)) | set(lay.rot_steps()))
    s = fhe.Session(ch, rot_steps=steps, k_max=4, seed=0, h=64, sigma=3.2, galois_extra=(BS.conj_galois(ch.n),))
    rng = np.random.default_rng(62)
    weights = [M.random_layer(rng, d=cfg.d, mlp=cfg.mlp, std=0.03) for _ in range(cfg.layers)]
    prompt = rng.normal(0, 1, (40, cfg.d))
    x = rng.normal(0, 1, cfg.d)
    dec = M.Decoder(s, cfg, weights, ch.q, BS.Bootstrapper(s, prm, ch.q, ch.q[0]))

    emb = torch.as_tensor(prompt, dtype=torch.float32, device="cuda")
    Ks, Vs, _ = PF.prefill(emb, [40], PF.load(weights, dtype=torch.float16), cfg)
    dec.load([K[0].cpu().double().numpy() for K in Ks], [V[0].cpu().double().numpy() for V in Vs])
    y = dec.decode(s.encrypt(LIN.input_vector(x, dec.lay.geo), 0, 2.0**40, dec.lay.slots))
    torch.cuda.synchronize()

    caches = [[np.zeros((0, cfg.d)), np.zeros((0, cfg.d))] for _ in weights]
    for tok in prompt:
        M.plain_decode(tok, weights, caches, cfg, dec.coeffs)
    want = M.plain_decode(x, weights, caches, cfg, dec.coeffs)
    got = LIN.output_values(s.decrypt_slots(y).real, dec.lay.geo, cfg.d)
    # the encrypted step's 1e-3 and the caches' 16-bit operands (tests/test_gpu_clear.py)
    assert np.abs(got - want).max() < 1e-3 + 16 * 2.0**-11
