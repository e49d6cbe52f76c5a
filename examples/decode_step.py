"""A small quantised decoder over the library: a prompt, then token after token from one captured CUDA graph.

Per layer: rms_norm (with the residual's addition), the fused q/k/v product, rope_append into the paged 8-bit cache,
attention over it, the output product, rms_norm, gate + up + SwiGLU, the down product; then the last norm, the logits
and sample. Weights are random Q4 tables. The captured step reads its lengths on the device: each replay makes the next
token of every sequence.

    python examples/decode_step.py [--layers 2] [--batch 4] [--prompt 100] [--tokens 32]
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "volta-kernel-bakeoff_b200"))
import vkb  # noqa: E402

HIDDEN, Q_HEADS, KV_HEADS, DIM, MLP, VOCAB, PAGE = 2048, 16, 2, 128, 6144, 32000, 64
QKV = (Q_HEADS + 2 * KV_HEADS) * DIM


def table(rows: int, cols: int, g) -> tuple:
    """A random Q4 table: packed codes and fp16 scales."""
    q = torch.randint(0, 256, (rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand((rows, cols // 32), generator=g, device="cuda") * 0.4 + 0.8) * (0.2 / cols ** 0.5)
    return q, s.half()


class Decoder:
    def __init__(self, layers: int, batch: int, longest: int, seed: int = 0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.batch = batch
        self.embed = torch.randn((VOCAB, HIDDEN), generator=g, device="cuda")
        self.layers = [dict(qkv=table(QKV, HIDDEN, g), out=table(HIDDEN, Q_HEADS * DIM, g), gate_up=table(2 * MLP, HIDDEN, g),
                            down=table(HIDDEN, MLP, g), norms=[torch.ones(HIDDEN, device="cuda").half() for _ in range(2)])
                       for _ in range(layers)]
        self.last_norm, self.head = torch.ones(HIDDEN, device="cuda").half(), table(VOCAB, HIDDEN, g)
        per = -(-longest // PAGE)
        self.caches = [vkb.KvCache.empty(per * batch, KV_HEADS, DIM, PAGE) for _ in range(layers)]
        # pages are handed out in turn: sequence b's page i is page i * batch + b
        self.pages = torch.arange(per * batch, device="cuda", dtype=torch.int32).view(per, batch).t().contiguous()
        self.turns, self.mscale = vkb.rope_turns(DIM, base=1e6)
        self.work = vkb.attention_workspace(self.caches[0])
        self.lens = torch.zeros(batch, device="cuda", dtype=torch.int32)      # lengths in the cache
        self.tokens = torch.zeros(batch, device="cuda", dtype=torch.int32)    # each sequence's next input
        self.u = torch.zeros(batch, device="cuda")
        self.settings = dict(temperature=torch.full((batch,), 0.8, device="cuda"), top_k=torch.full((batch,), 50, device="cuda", dtype=torch.int32),
                             top_p=torch.full((batch,), 0.95, device="cuda"))

    @staticmethod
    def product(w, x):
        """x . W^T: the decode kernel up to 8 rows, the tensor-core kernel for more."""
        return vkb.gemv(vkb.FMT_Q4, *w, x) if x.shape[0] <= 8 else vkb.gemm_tc(*w, x)

    def mlp(self, w, x):
        if x.shape[0] <= 8:
            return vkb.gate_up_glu_q4(*w, x, out_f32=False, want_stack=False)[0]
        gate, up = self.product(w, x).float().chunk(2, -1)
        return (torch.nn.functional.silu(gate) * up).half()

    def forward(self, tokens, cu=None):
        """Hidden states [rows][HIDDEN] of the tokens appended to the sequences; self.lens already counts them. cu: row
        offsets (None: one token per sequence)."""
        stream = self.embed[tokens.long()]                        # the residual stream, fp32
        branch = stream.half() * 0
        for layer, cache in zip(self.layers, self.caches):
            x, stream, *_ = vkb.rms_norm(branch, layer["norms"][0], stream)
            qkv = self.product(layer["qkv"], x).view(-1, Q_HEADS + 2 * KV_HEADS, DIM)
            q, k, v = qkv[:, :Q_HEADS], qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], qkv[:, Q_HEADS + KV_HEADS:]
            q = vkb.rope_append(cache, self.pages, self.lens, q, k, v, turns=self.turns, mscale=self.mscale, cu=cu)
            a = vkb.attention(cache, self.pages, self.lens, q, cu=cu, work=self.work)
            branch = self.product(layer["out"], a.view(-1, Q_HEADS * DIM))
            x, stream, *_ = vkb.rms_norm(branch, layer["norms"][1], stream)
            branch = self.product(layer["down"], self.mlp(layer["gate_up"], x))
        return vkb.rms_norm(branch, self.last_norm, stream)[0]

    def logits(self, x):
        return torch.cat([vkb.gemv(vkb.FMT_Q4, *self.head, part, out_f32=True) for part in x.split(8)])

    def prompt(self, prompts):
        """Take in a list of 1-D int32 token tensors; the logits of each one's last token."""
        news = [len(p) for p in prompts]
        cu = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], device="cuda", dtype=torch.int32)
        self.lens += torch.tensor(news, device="cuda", dtype=torch.int32)
        x = self.forward(torch.cat(prompts), cu)
        return self.logits(x[cu[1:].long() - 1])

    def step(self):
        """One token per sequence: self.tokens goes in, and the sampled next one takes its place."""
        self.lens += 1
        logits = self.logits(self.forward(self.tokens))
        vkb.sample(logits, self.u, token=self.tokens, **self.settings)
        return logits


def run(layers=2, batch=4, prompt=100, tokens=32, seed=0):
    """Generated tokens [tokens][batch] and the decoder."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    d = Decoder(layers, batch, prompt + tokens + 8, seed)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    made = []
    with torch.cuda.stream(stream):
        logits = d.prompt([torch.randint(0, VOCAB, (max(1, prompt - 7 * b),), generator=g, device="cuda", dtype=torch.int32) for b in range(batch)])
        vkb.sample(logits, torch.rand(batch, generator=g, device="cuda"), token=d.tokens, **d.settings)
        made.append(d.tokens.clone())
        d.u.copy_(torch.rand(batch, generator=g, device="cuda"))
        d.step()                                  # a first step outside the graph: what is set up once is set up
        made.append(d.tokens.clone())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            d.step()
        for _ in range(tokens - 2):
            d.u.copy_(torch.rand(batch, generator=g, device="cuda"))
            graph.replay()
            made.append(d.tokens.clone())
    stream.synchronize()
    return torch.stack(made), d


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("layers", 2), ("batch", 4), ("prompt", 100), ("tokens", 32)):
        ap.add_argument("--" + name, type=int, default=default)
    made, d = run(**vars(ap.parse_args()))
    status = vkb.device_status()
    print("lengths", d.lens.tolist())
    for b in range(d.batch):
        print("sequence", b, made[:, b].tolist())
    sys.exit(1 if status else 0)
