"""Batched greedy generation over a paged 4-bit KV cache: the operators of
``bfp200.kv4`` together, in the layer of the reference simulator (fwd_layer,
gen_smollm_blockfp_full.py:261-293).

    python -m bfp200.paged --layers 2 --seqs 4 --n-gen 8

Matrices, norms and quantization are the framework's BFP operators; positions,
cache and attention are kv4's, so unlike the Decoder's stream this one carries
the rounding of 4-bit keys and values (6,480 bytes a position of the 30-layer
model instead of 23,760).  Prompts of any length enter in one call, sequences
hold only the pages that they use, and the rotation table may be a scaled one.
Each step feeds the argmax of the one before.  The head runs on the host: this
shows how the operators fit together, not the fastest decode of a small model.
"""
from __future__ import annotations

import numpy as np
import torch

from . import kv4, ops
from .config import BfpConfig


class PagedDecoder:
    """One synthetic-format model (see synth.synthetic_model) and its caches."""

    def __init__(self, cfg: BfpConfig, model, n_pages, page=16, table=None, max_pos=None, device=None):
        self.cfg, self.page = cfg, page
        self.layers, g1, g2, self.embed, nw = model
        self.g1, self.g2 = [ops.tile_decode(*g) for g in g1], [ops.tile_decode(*g) for g in g2]
        self.norm_w = ops.tile_decode(*nw)
        self.emb = ops.tile_decode(self.embed[0].reshape(-1), self.embed[1].reshape(-1)).reshape(cfg.VOCAB, cfg.D)
        self.device = device or torch.device("cuda")
        self.pools = [kv4.new_pool(n_pages, cfg.H_KV, cfg.HD, page, self.device) for _ in range(cfg.NL)]
        self.table = kv4.rope_table(max_pos or cfg.MAX_CTX, cfg.HD, cfg.rope_base, device=self.device) if table is None else table
        self.free = list(range(n_pages))[::-1]

    def _matvec(self, x, w):
        """The BFP matvec of rows x [T, D] on the grid."""
        m, e = ops.tile_quantize(x)
        t, d = x.shape
        om, oe = ops.matvec(m.reshape(t, d // 16, 16), e.reshape(t, d // 16), *w)
        return ops.tile_decode(om.reshape(-1), oe.reshape(-1)).reshape(t, -1)

    @staticmethod
    def _grid(x):
        return ops.fp_quantize_vec(x).reshape(x.shape)

    def _gpu(self, x, heads):
        return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(self.device).view(len(x), heads, self.cfg.HD)

    def forward(self, tokens, q_start, lens, block_table):
        """Logits [T, VOCAB] (float64) of the call's tokens; appends them to the cache."""
        cfg = self.cfg
        h = self.emb[np.asarray(tokens)]
        for i, lw in enumerate(self.layers):
            n1 = ops.rmsnorm_fp(h, self.g1[i], cfg.eps)
            q, k, v = (self._gpu(self._matvec(n1, lw[w]), n) for w, n in (("Wq", cfg.H_Q), ("Wk", cfg.H_KV), ("Wv", cfg.H_KV)))
            q = kv4.append(self.pools[i], k, v, q_start, lens, block_table, q=q, table=self.table)
            attn = kv4.attention(q, self.pools[i], q_start, lens, block_table, check_done=True)
            h = self._grid(h + self._matvec(attn.view(len(h), -1).double().cpu().numpy(), lw["Wo"]))
            n2 = ops.rmsnorm_fp(h, self.g2[i], cfg.eps)
            mlp = ops.silu_fp(self._matvec(n2, lw["Wg"])) * self._matvec(n2, lw["Wu"])
            h = self._grid(h + self._matvec(mlp, lw["Wd"]))
        return ops.rmsnorm_fp(h, self.norm_w, cfg.eps) @ self.emb.T

    def generate(self, prompts, n_gen):
        """prompt + n_gen greedy ids per sequence (of no sequences, none)."""
        lens = [len(p) for p in prompts]
        if not lens:
            return []
        if min(lens) < 1:
            raise ValueError("a prompt needs at least one id")
        need = [-(-(n + n_gen) // self.page) for n in lens]
        if sum(need) > len(self.free):
            raise ValueError(f"{sum(need)} pages are needed, {len(self.free)} are free")
        if self.page * max(need) > self.table.shape[0]:
            raise ValueError("the rotation table is shorter than the longest sequence's pages")
        table = np.zeros((len(prompts), max(need)), np.int32)
        for s, n in enumerate(need):
            table[s, :n] = [self.free.pop() for _ in range(n)]
        bt = torch.from_numpy(table).to(self.device)
        out = [list(p) for p in prompts]
        ints = lambda a: torch.tensor(a, dtype=torch.int32, device=self.device)
        try:
            new = [list(p) for p in prompts]
            for _ in range(n_gen):
                starts = np.concatenate([[0], np.cumsum([len(x) for x in new])])
                logits = self.forward(np.concatenate(new), ints(starts), ints(lens), bt)
                for s, last in enumerate(starts[1:] - 1):
                    out[s].append(int(np.argmax(logits[last])))
                new = [[o[-1]] for o in out]
                lens = [n + 1 for n in lens]
        finally:
            for s, n in enumerate(need):
                self.free += table[s, :n].tolist()
        return out


def main(argv=None):
    import argparse
    from . import synth
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=2048)
    ap.add_argument("--seqs", type=int, default=4)
    ap.add_argument("--n-gen", type=int, default=8)
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--scaling", choices=kv4.SCALINGS, default="none")
    ap.add_argument("--factor", type=float, default=1.0)
    a = ap.parse_args(argv)
    cfg = BfpConfig(NL=a.layers, VOCAB=a.vocab)
    rng = np.random.default_rng(3)
    prompts = [rng.integers(0, a.vocab, int(n)).tolist() for n in rng.integers(8, 49, a.seqs)]
    most = max(map(len, prompts)) + a.n_gen
    pages = sum(-(-(len(p) + a.n_gen) // a.page) for p in prompts)
    table = kv4.rope_table(-(-most // a.page) * a.page, cfg.HD, cfg.rope_base, a.scaling, a.factor)
    dec = PagedDecoder(cfg, synth.synthetic_model(cfg), pages, a.page, table)
    for s, ids in enumerate(dec.generate(prompts, a.n_gen)):
        print(f"sequence {s}: {len(prompts[s])} prompt ids ->", *ids[len(prompts[s]):])
    print(f"cache: {sum(p.numel() for p in dec.pools)} bytes in {pages} pages of {a.page} positions and {a.layers} layers")


if __name__ == "__main__":
    main()
