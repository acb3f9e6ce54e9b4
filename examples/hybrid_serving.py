"""A small hybrid model served from its caches: KDA layers with their
recurrent states, every fourth layer softmax attention over a paged cache.

    python examples/hybrid_serving.py        # needs a ROCm GPU

Prompts of uneven lengths are prefilled packed, each is continued token by
token, beams are forked and freed, the pool is compacted, and decoding goes
on.  Weights are random: what runs is the path of a serving loop, not a
language model.  :class:`Server` keeps

* ``states`` ``[KDA layers, rows, H, 128, 128]`` fp32: a recurrent state for
  each row and KDA layer;
* ``pool`` ``[attention layers, 2, pages, HKV, page_size, 128]`` bf16: keys
  and values, the tokens of a head together;
* ``table``, ``lens``, ``refs``: the pages of each row, its cached tokens, the
  holders of each page (:mod:`kda_bt16.paged`).
"""

from __future__ import annotations

import sys
from pathlib import Path

import torch
import torch.nn.functional as F

_PKG = Path(__file__).resolve().parents[1] / "kda-ascendc_amd"
if str(_PKG) not in sys.path:
    sys.path.insert(0, str(_PKG))

import kda_bt16  # noqa: E402

D = 128
PAGE = 16
LOWER_BOUND = -5.0


class Model:
    """Random weights: ``layers`` layers, every fourth one attention with HQ
    query and HKV key heads, the others KDA with H heads."""

    def __init__(self, layers=8, hidden=512, H=4, HQ=8, HKV=2, vocab=1000, device="cuda", seed=0):
        gen = torch.Generator(device=device).manual_seed(seed)

        def w(*shape):
            return (torch.randn(*shape, generator=gen, device=device) * shape[0] ** -0.5).bfloat16()

        self.H, self.HQ, self.HKV, self.hidden, self.vocab = H, HQ, HKV, hidden, vocab
        self.embed = w(vocab, hidden) * vocab ** 0.5
        self.head = w(hidden, vocab)
        self.layers = []
        for i in range(layers):
            if i % 4 == 3:
                self.layers.append({"kind": "attention", "qkv": w(hidden, (HQ + 2 * HKV) * D), "out": w(HQ * D, hidden)})
            else:
                self.layers.append({
                    "kind": "kda", "qkvg": w(hidden, 4 * H * D), "beta": w(hidden, H), "out": w(H * D, hidden),
                    "A_log": torch.log(1.0 + 15.0 * torch.rand(H, generator=gen, device=device)),
                    "dt_bias": 0.1 * torch.randn(H * D, generator=gen, device=device),
                })

    def count(self, kind):
        return sum(x["kind"] == kind for x in self.layers)


class Server:
    def __init__(self, model: Model, rows=8, pages=64, max_tokens=512, device="cuda"):
        self.m, self.rows, self.device = model, rows, device
        self.states = torch.zeros(model.count("kda"), rows, model.H, D, D, device=device)
        self.pool = torch.zeros(model.count("attention"), 2, pages, model.HKV, PAGE, D, dtype=torch.bfloat16,
                                device=device)
        self.table = torch.full((rows, -(-max_tokens // PAGE)), -1, dtype=torch.int32, device=device)
        self.lens = torch.zeros(rows, dtype=torch.int32, device=device)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=device)

    def _rows(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.device)

    def _reserve(self, more):
        ok = kda_bt16.paged_reserve(self.table, self.lens, self.refs, self._rows(more), PAGE)
        if not bool(ok.all()):
            raise RuntimeError("the pool is out of pages")

    def _layers(self, x, cu):
        """x [B, T, hidden] through all layers; cu: packed prompts, one a row
        (fresh states), else one token of every row."""
        m, kda_i, attn_i = self.m, 0, 0
        B, T = x.shape[:2]
        for layer in m.layers:
            h = F.rms_norm(x, (m.hidden,))
            if layer["kind"] == "kda":
                q, k, v, g = (t.contiguous() for t in (h @ layer["qkvg"]).view(B, T, 4, m.H, D).unbind(2))
                kw = dict(use_qk_l2norm_in_kernel=True, use_gate_in_kernel=True, use_beta_sigmoid_in_kernel=True,
                          lower_bound=LOWER_BOUND, A_log=layer["A_log"], dt_bias=layer["dt_bias"], state_v_first=True)
                beta = h @ layer["beta"]
                if cu is None:
                    o = kda_bt16.kda_decode_step(q, k, v, g, beta, self.states[kda_i], **kw)
                else:
                    o, last = kda_bt16.chunk_kda(q, k, v, g, beta, output_final_state=True, safe_gate=True, cu_seqlens=cu,
                                                 **kw)
                    self.states[kda_i] = last
                kda_i += 1
            else:
                qkv = (h @ layer["qkv"]).view(B, T, m.HQ + 2 * m.HKV, D)
                q, k, v = qkv.split([m.HQ, m.HKV, m.HKV], 2)
                # [pages, tokens, heads, D] views of the heads' tokens
                kc, vc = self.pool[attn_i, 0].transpose(1, 2), self.pool[attn_i, 1].transpose(1, 2)
                kda_bt16.paged_append(k, v, kc, vc, self.table, self.lens, cu_seqlens=cu)
                o = kda_bt16.paged_attention(q, kc, vc, self.table, self.lens, cu_seqlens=cu)
                attn_i += 1
            x = x + o.reshape(B, T, -1) @ layer["out"]
        return F.rms_norm(x, (m.hidden,)) @ m.head

    def prefill(self, prompts):
        """One prompt (a list of tokens) a row, into empty rows; the logits
        after each one's last token."""
        lens = [len(x) for x in prompts]
        self._reserve(lens)
        cu = self._rows([0] + lens).cumsum(0, dtype=torch.int32)
        tokens = torch.tensor([t for x in prompts for t in x], device=self.device)
        logits = self._layers(self.m.embed[tokens][None], cu)
        return logits[0, (cu[1:] - 1).long()]

    def step(self, tokens):
        """One more token of every row; the logits after it."""
        self._reserve([1] * self.rows)
        return self._layers(self.m.embed[tokens][:, None], None)[:, 0]

    def fork(self, src, dst):
        """Rows dst end; they go on as copies of rows src."""
        src, dst = self._rows(src), self._rows(dst)
        kda_bt16.paged_free(self.table, self.lens, self.refs, dst)
        ok = kda_bt16.paged_fork(self.pool, self.table, self.lens, self.refs, src, dst, page_size=PAGE)
        if not bool(ok.all()):
            raise RuntimeError("the pool is out of pages")
        kda_bt16.paged_copy(self.states, src, dst)

    def compact(self):
        """The held pages become the pool's first; their number."""
        self.table, self.refs, live = kda_bt16.paged_compact(self.pool, self.table, self.refs)
        return int(live)


def main():
    torch.manual_seed(0)
    model = Model()
    server = Server(model, rows=4)
    prompts = [torch.randint(0, model.vocab, (n,)).tolist() for n in (37, 5, 64, 120)]
    texts = [list(x) for x in prompts]
    logits = server.prefill(prompts)
    for step in range(20):
        tokens = logits.argmax(-1)
        for row, t in enumerate(tokens.tolist()):
            texts[row].append(t)
        logits = server.step(tokens)
        if step == 9:
            # row 1 ends, row 2 goes on twice
            server.fork([2], [1])
            texts[1], logits[1] = list(texts[2]), logits[2]
            print("pages held after compaction:", server.compact(), flush=True)
    print("tokens cached:", server.lens.tolist())
    for row, text in enumerate(texts):
        print(f"row {row}: {len(text)} tokens, the last of them {text[-8:]}")


if __name__ == "__main__":
    main()
