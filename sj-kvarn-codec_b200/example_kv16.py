"""Parallel samples of one prompt on a small random model whose layers are partly kept at 16 bits and partly sealed:
the calls of kv16 together as a server would make them.

    python example_kv16.py [--samples 4] [--prompt 300] [--steps 40]

Per layer and step: one sjk_qkv (norm, rotary positions, cache write or 32-bit rows), then sjk_kv16_attend over the
pages, or sjk_store_batch and sjk_attend_batch over sealed caches. The prompt is prefilled once; its pages are shared by
the samples (fork), split when a sample writes on (extend), given back when it ends (free), and the pool is compacted.
"""
import argparse
import ctypes as C
import math

import torch

import kv16
import sjk

DIM, HEADS, HEADS_KV, D, VOCAB = 256, 8, 2, 128, 199
PAGE = 16


class Model:
    """Random weights; kinds: "kv16" or "sealed" for every layer."""

    def __init__(self, kinds=("kv16", "sealed", "kv16"), seed=0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        rand = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
        self.kinds = kinds
        self.embed = rand(VOCAB, DIM)
        self.wqkv = [rand(DIM, (HEADS + 2 * HEADS_KV) * D) / math.sqrt(DIM) for _ in kinds]
        self.wo = [rand(HEADS * D, DIM) / math.sqrt(HEADS * D) for _ in kinds]
        self.norms = [(1 + 0.1 * rand(D), 1 + 0.1 * rand(D)) for _ in kinds]
        self.rope = kv16.Rope(D, base=1e5)

    def heads(self, il, x):
        """q, k, v of rows x as bf16 views of one projection."""
        n = x.shape[0]
        y = (x @ self.wqkv[il]).bfloat16()
        return [y[:, a * D: b * D].view(n, b - a, D) for a, b in
                ((0, HEADS), (HEADS, HEADS + HEADS_KV), (HEADS + HEADS_KV, HEADS + 2 * HEADS_KV))]


class Server:
    """Caches of `slots` sequences of up to `ctx` tokens; row 0 is the prompt's."""

    def __init__(self, model, slots, ctx):
        self.m, self.slots, self.L = model, slots, sjk.lib()
        stride = -(-ctx // PAGE)
        self.at = {il: i for i, il in enumerate(i for i, k in enumerate(model.kinds) if k == "kv16")}     # cache layers
        self.cache = kv16.Cache.alloc(max(len(self.at), 1), (slots + 1) * stride, PAGE, HEADS_KV, D, torch.bfloat16, slots, stride)
        self.pages = self.cache.pages()
        self.steps = [kv16.Qkv(D, rope=model.rope, q_norm=a, k_norm=b, cache=self.cache if k == "kv16" else None)
                      for k, (a, b) in zip(model.kinds, model.norms)]
        # sealed layers: a cache per sequence, whose staging ring holds all of it (nothing is sealed in so short a run)
        tail = -(-ctx // 128) * 128
        cfg = sjk.config(D, HEADS_KV, 2 * tail + 512, 512, tail=tail, tail_max=2 * tail)
        self.cfg = cfg
        self.sealed = {il: [sjk.Layer() for _ in range(slots)] for il, k in enumerate(model.kinds) if k == "sealed"}
        for layers in self.sealed.values():
            for x in layers:
                sjk.check(self.L.sj_kvarn_layer_init(C.byref(x), C.byref(cfg)), "layer_init")
        self.views = {il: (sjk.View * slots)(*[sjk.view_of(x) for x in layers]) for il, layers in self.sealed.items()}
        self.scale = 1 / math.sqrt(D)

    def close(self):
        torch.cuda.synchronize()
        for layers in self.sealed.values():
            for x in layers:
                self.L.sj_kvarn_layer_free(C.byref(x))

    def _stream(self):
        return torch.cuda.current_stream().cuda_stream

    def prefill(self, tokens):
        """The prompt's cache rows in sequence 0 (every sealed cache gets its own). The layers' inputs are the tokens'
        embeddings: the toy has no attention within the prompt."""
        n = tokens.shape[0]
        row0 = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.pages.extend(row0, row0, n)
        x = self.m.embed[tokens]
        pos = torch.arange(n, dtype=torch.int32, device="cuda")
        for il, kind in enumerate(self.m.kinds):
            q, k, v = self.m.heads(il, x)
            if kind == "kv16":
                self.steps[il](k=k, v=v, pos=pos, rows=torch.zeros(n, dtype=torch.int32, device="cuda"), layer=self.at[il])
            else:
                kr, vr = (torch.empty((n, HEADS_KV, D), dtype=torch.float32, device="cuda") for _ in range(2))
                self.steps[il](k=k, v=v, pos=pos, k_out=kr, v_out=vr)
                for layer in self.sealed[il]:
                    sjk.check(self.L.sjk_layer_store(C.byref(layer), 0, n, kr.data_ptr(), vr.data_ptr(), 1, self._stream()), "layer_store")

    def fork(self, n):
        """Sequences 1 .. n - 1 share the prompt's pages."""
        dst = torch.arange(1, n, dtype=torch.int32, device="cuda")
        return self.pages.fork(torch.zeros_like(dst), dst)

    def step(self, tokens, length):
        """One token for each of the sequences 0 .. n - 1, all of `length` tokens so far: their logits."""
        n = tokens.shape[0]
        rows = torch.arange(n, dtype=torch.int32, device="cuda")
        lens = torch.full((n,), length, dtype=torch.int32, device="cuda")
        self.pages.extend(rows, lens, 1)
        x = self.m.embed[tokens]
        for il, kind in enumerate(self.m.kinds):
            q, k, v = self.m.heads(il, x)
            if kind == "kv16":
                q2 = torch.empty((n, HEADS, D), dtype=torch.bfloat16, device="cuda")
                self.steps[il](q, k, v, lens, q_out=q2, rows=rows, layer=self.at[il])
                att = self.cache.attend(self.at[il], q2, lens + 1, self.scale, rows=rows, out=torch.empty_like(q2, dtype=torch.float32))
            else:
                q2 = torch.empty((n, HEADS, D), dtype=torch.float32, device="cuda")
                kr, vr = (torch.empty((n, HEADS_KV, D), dtype=torch.float32, device="cuda") for _ in range(2))
                self.steps[il](q, k, v, lens, q_out=q2, k_out=kr, v_out=vr)
                att = self._sealed(il, n, length, q2, kr, vr)
            x = x + att.reshape(n, -1) @ self.m.wo[il]
        return x @ self.m.embed.T

    def _sealed(self, il, n, length, q, k, v):
        st, u32 = self._stream(), C.c_uint32 * n
        sjk.check(self.L.sjk_store_batch(self.views[il], u32(*[length] * n), n, k.data_ptr(), v.data_ptr(), 1, st), "store_batch")
        sjk.check(self.L.sjk_hadamard(q.data_ptr(), n * HEADS, D, st), "hadamard")
        out = torch.empty_like(q)
        size = self.L.sjk_attend_batch_scratch_bytes(C.byref(self.views[il][0]), n, 1, HEADS)
        scratch = torch.empty(size, dtype=torch.uint8, device="cuda")
        S = self.cfg.sink
        sjk.check(self.L.sjk_attend_batch(self.views[il], u32(*[S] * n), u32(*[length + 1] * n), u32(*[length] * n), n, 1, HEADS,
                                          q.data_ptr(), self.scale, out.data_ptr(), scratch.data_ptr(), size, st), "attend_batch")
        sjk.check(self.L.sjk_hadamard(out.data_ptr(), n * HEADS, D, st), "hadamard")
        return out

    def finish(self, n):
        """Sequences 1 .. n - 1 end; their pages go back and the used ones to the front of the pool."""
        self.pages.free(torch.arange(1, n, dtype=torch.int32, device="cuda"))
        return self.pages.compact()


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--samples", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=40)
    a = ap.parse_args()
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    s = Server(Model(), a.samples, a.prompt + a.steps + PAGE)
    s.prefill(torch.randint(0, VOCAB, (a.prompt,), device="cuda", generator=g))
    s.fork(a.samples)
    free = s.pages.n_free.item()
    tokens = torch.randint(0, VOCAB, (a.samples,), device="cuda", generator=g)
    chosen = []
    for i in range(a.steps):
        p = torch.softmax(s.step(tokens, a.prompt + i) / math.sqrt(DIM), -1)
        tokens = torch.multinomial(p, 1, generator=g)[:, 0]
        chosen.append(tokens)
    for i, row in enumerate(torch.stack(chosen, 1).tolist()):
        print(f"sample {i}: {row[:16]} ...")
    print(f"{a.samples} samples of {a.prompt} + {a.steps} tokens took {free - s.pages.n_free.item()} pages beside the prompt's")
    print(f"after the samples ended: {s.finish(a.samples).tolist()} (used pages, moved)")
    assert s.L.sjk_device_status() == 0
    s.close()


if __name__ == "__main__":
    main()
