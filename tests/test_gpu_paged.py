"""Generation over the paged 4-bit cache (bfp200.paged) against the same loop
in 64 bits: the oracle's BFP layer with keys and values rounded to 4-bit tiles
and attention from its formula.  Hidden values are re-quantized to 16-bit tiles
after every sum, so the two runs' logits may differ by roundings of 2^-15 that
went the other way; the argmax has to agree."""
import numpy as np
import pytest

from oracle import bfp_oracle as B, kv4_oracle as K

pytestmark = pytest.mark.gpu


def _oracle_generate(cfg, model, prompts, n_gen):
    layers, g1, g2, embed, nw = model
    dec = lambda me: B.tile_decode(np.asarray(me[0]).reshape(-1), np.asarray(me[1]).reshape(-1))
    emb = dec(embed).reshape(cfg.VOCAB, cfg.D)
    ocfg = B.Cfg(D=cfg.D, H_Q=cfg.H_Q, H_KV=cfg.H_KV, HD=cfg.HD, FFN=cfg.FFN, NL=cfg.NL, VOCAB=cfg.VOCAB)
    f = 10000.0 ** (-np.arange(0, cfg.HD, 2) / cfg.HD)
    outs = []
    for p in prompts:
        ids, kv = list(p), [([], []) for _ in layers]
        for step in range(len(p) + n_gen - 1):
            h = emb[ids[step]]
            a = step * f
            cs = np.stack([np.cos(a), np.sin(a)], -1).astype(np.float32)[None]
            for (ks, vs), lw, ga, gb in zip(kv, layers, g1, g2):
                mv = lambda x, w: B.matvec_cols(*(y[None] for y in B.tile_quantize(x)), *lw[w])[0]
                n1 = B.rmsnorm_fp(h, dec(ga), cfg.eps)
                q, k, v = (mv(n1, w).reshape(1, -1, cfg.HD) for w in ("Wq", "Wk", "Wv"))
                q, k = (K.rotate32(x, cs, cfg.HD, False).astype(np.float64) for x in (q, k))
                ks.append(K.value(*K.quantize(k[0])))
                vs.append(K.value(*K.quantize(v[0].astype(np.float32))))
                n = len(ks)
                attn = K.attention(q, np.array(ks), np.array(vs), K.visible(n, 1, True, 0), cfg.HD ** -0.5)[0].reshape(-1)
                h = B.fp_quantize_vec(h + mv(attn, "Wo"))
                n2 = B.rmsnorm_fp(h, dec(gb), cfg.eps)
                h = B.fp_quantize_vec(h + mv(B.silu_fp(mv(n2, "Wg")) * mv(n2, "Wu"), "Wd"))
            if step >= len(p) - 1:
                ids.append(int(np.argmax(B.rmsnorm_fp(h, dec(nw), cfg.eps) @ emb.T)))
        outs.append(ids)
    return outs


@pytest.mark.parametrize("heads,page", [((3, 1), 16), ((2, 2), 32)])
def test_paged_generation(heads, page):
    from bfp200 import BfpConfig, paged, synth
    cfg = BfpConfig(D=64 * heads[0], H_Q=heads[0], H_KV=heads[1], FFN=128, NL=2, VOCAB=256, MAX_CTX=64)
    model = synth.synthetic_model(cfg, seed=5)
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, cfg.VOCAB, n).tolist() for n in (1, 17, 5, 33)]
    dec = paged.PagedDecoder(cfg, model, n_pages=12, page=page)
    got = dec.generate(prompts, 6)
    assert got == _oracle_generate(cfg, model, prompts, 6)
    assert sorted(dec.free) == list(range(12))                # every page came back
    assert dec.generate(prompts[::-1], 6) == got[::-1]        # other pages, other order: the same tokens


def test_paged_refusals():
    from bfp200 import BfpConfig, paged, synth
    cfg = BfpConfig(D=64, H_Q=1, H_KV=1, FFN=64, NL=1, VOCAB=64, MAX_CTX=32)
    dec = paged.PagedDecoder(cfg, synth.synthetic_model(cfg, seed=1), n_pages=2, page=16)
    with pytest.raises(ValueError):
        dec.generate([[1] * 30], 8)                            # three pages
    dec = paged.PagedDecoder(cfg, synth.synthetic_model(cfg, seed=1), n_pages=4, page=16)
    with pytest.raises(ValueError):
        dec.generate([[1] * 30], 8)                            # past the rotation table
    assert len(dec.free) == 4


def test_paged_command(capsys):
    from bfp200 import paged
    paged.main(["--layers", "1", "--vocab", "256", "--seqs", "2", "--n-gen", "3", "--scaling", "bands", "--factor", "2"])
    out = capsys.readouterr().out
    assert out.count("sequence ") == 2 and "bytes in" in out
