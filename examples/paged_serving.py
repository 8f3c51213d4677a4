"""Requests served together from one pool of pages with 4-bit keys and values.

A step takes the next rows of every request that has a slot: a chunk of a
prompt, or the one token picked last. The rows go through the layers side by
side; si_paged_rope_kv_append stores their keys and values in the requests'
pages, si_paged_attention reads them, and si_process_logits applies each
request's penalties, biases and grammar mask to its logits and picks the next
token. Pages are taken from a free list as requests grow and go back when they
end. A waiting request takes a slot that became free once the pool has room for
it at its full length, beside those that are being served.

    python examples/paged_serving.py [--requests 6] [--slots 4] [--tokens 24]
"""
from __future__ import annotations

import argparse
import ctypes as C
import sys
from dataclasses import dataclass, field
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from sharpinference_b200 import native, phi4  # noqa: E402


@dataclass
class Request:
    prompt: np.ndarray                  # token ids
    new_tokens: int
    repetition: float = 1.0
    frequency: float = 0.0
    presence: float = 0.0
    biases: dict = field(default_factory=dict)
    allowed: np.ndarray | None = None   # bool [vocab]: the grammar's tokens
    tokens: list = field(default_factory=list)  # picked so far

    def __post_init__(self):
        self.held = 0  # tokens whose keys and values are in the cache

    @property
    def done(self):
        return len(self.tokens) >= self.new_tokens

    def next_rows(self, chunk):
        """The tokens that are not in the cache yet, a chunk of them at most."""
        every = np.concatenate([self.prompt, np.asarray(self.tokens, np.int32)])
        return every[self.held:self.held + chunk]


class PagedServer:
    """`weights`: the decoder session's slots (native.decoder_slot_names) as host arrays of GGUF bytes, norms as
    float32; the embedding has to be F16."""

    def __init__(self, cfg, weights, slots, pages, page_size=64, chunk=512):
        if cfg["embedding_type"] != native.F16:
            raise native.ArgumentError("the batched embedding lookup takes an F16 table.")
        self.cfg, self.slots, self.pages, self.page_size, self.chunk = cfg, slots, pages, page_size, chunk
        self.weights = {n: torch.from_numpy(np.array(w)).cuda() for n, w in weights.items()}
        rotary = cfg["rotary_size"]
        self.frequencies = torch.from_numpy(
            (cfg["rope_base"] ** (-np.arange(0, rotary, 2) / rotary)).astype(np.float32)).cuda()
        kv, d = cfg["kv_heads"], cfg["head_size"]
        bytes_of_layer = native.paged_cache_bytes(pages, page_size, kv, d)
        self.pool = torch.zeros(cfg["layers"], bytes_of_layer, dtype=torch.uint8, device="cuda")
        self.width = (cfg["context"] + page_size - 1) // page_size
        self.table = np.full((slots, self.width), -1, np.int32)
        self.device_table = torch.from_numpy(self.table).cuda()
        # one table for all layers, whose pages lie in pools of their own
        self.caches = [native.PagedCache(self.pool[layer].data_ptr(), self.device_table.data_ptr(), pages, slots,
                                         self.width, page_size, kv, d) for layer in range(cfg["layers"])]
        self.free = list(range(pages))
        self.active: list[Request | None] = [None] * slots
        self.waiting: list[Request] = []
        need = native.paged_attention_workspace_bytes(self.caches[0], slots * chunk, chunk, cfg["query_heads"])
        self.workspace = torch.zeros(need, dtype=torch.uint8, device="cuda")

    def submit(self, request: Request):
        if request.new_tokens < 1 or not 0 < len(request.prompt) <= self.cfg["context"] - request.new_tokens:
            raise native.ArgumentError("a request's tokens have to fit the context.")
        if self._pages(request) > self.pages:
            raise native.ArgumentError("a request's tokens have to fit the pool.")
        self.waiting.append(request)

    def run(self):
        """Steps until every request is done."""
        while any(self.active) or self.waiting:
            self.step()

    # ---- pages ---------------------------------------------------------------------------
    def _pages(self, request):
        """Pages of a request at its full length; the token picked last is never written."""
        return (len(request.prompt) + request.new_tokens - 1 + self.page_size - 1) // self.page_size

    def _admit(self):
        for slot in range(self.slots):
            if self.active[slot] is None and self.waiting:
                taken = sum(self._pages(r) for r in self.active if r)
                if taken + self._pages(self.waiting[0]) > self.pages:
                    return
                self.active[slot] = self.waiting.pop(0)

    def _grow(self, slot, tokens):
        for page in range((tokens + self.page_size - 1) // self.page_size):
            if self.table[slot, page] < 0:
                self.table[slot, page] = self.free.pop()

    def _release(self, slot):
        self.free += [int(p) for p in self.table[slot] if p >= 0]
        self.table[slot] = -1
        self.active[slot] = None

    # ---- one step ------------------------------------------------------------------------
    def step(self):
        self._admit()
        rows = [r.next_rows(self.chunk) if r else np.empty(0, np.int32) for r in self.active]
        lengths = [r.held + len(t) if r else 0 for r, t in zip(self.active, rows)]
        for slot, r in enumerate(self.active):
            if r:
                self._grow(slot, lengths[slot])
        self.device_table.copy_(torch.from_numpy(self.table))
        starts = np.concatenate([[0], np.cumsum([len(t) for t in rows])]).astype(np.int32)
        logits = self._forward(np.concatenate(rows).astype(np.int32), starts, np.asarray(lengths, np.int32))
        # requests whose last token's logits these are
        ready = [s for s, r in enumerate(self.active) if r and lengths[s] == len(r.prompt) + len(r.tokens)]
        for slot, r in enumerate(self.active):
            if r:
                r.held = lengths[slot]
        if not ready:
            return
        last = torch.from_numpy(starts[1:][ready].astype(np.int64) - 1).cuda()
        picked = self._pick(logits(last), [self.active[s] for s in ready])
        for slot, token in zip(ready, picked):
            request = self.active[slot]
            request.tokens.append(int(token))
            if request.done:
                self._release(slot)

    def _forward(self, tokens, starts, lengths):
        """Rows of all slots through the layers; returns a function of row indices that gives their logits."""
        cfg, w, stream = self.cfg, self.weights, torch.cuda.current_stream().cuda_stream
        rows, hidden, heads, kv, d = len(tokens), cfg["hidden"], cfg["query_heads"], cfg["kv_heads"], cfg["head_size"]
        most = int(max(np.diff(starts)))
        ids, starts, lengths = (torch.from_numpy(x).cuda() for x in (tokens, starts, lengths))
        control = torch.tensor([0, rows], dtype=torch.int32, device="cuda")

        def buffer(columns):
            return torch.empty(rows, columns, device="cuda")

        def project(name, x, wt=cfg["weight_type"]):
            width = {"qkv": hidden + 2 * kv * d, "attn_output": hidden, "ffn_up": 2 * cfg["intermediate"],
                     "ffn_down": hidden}[name.split("_weight_")[0]]
            y = buffer(width)
            native.call("si_batch_shared_matvec", wt, w[name].data_ptr(), x.data_ptr(), control.data_ptr(), y.data_ptr(),
                        rows, width, x.shape[1], stream)
            return y

        h, normed = buffer(hidden), buffer(hidden)
        native.call("si_embedding_gather_batch", w["token_embedding"].data_ptr(), cfg["vocab"], ids.data_ptr(),
                    h.data_ptr(), rows, hidden, stream)
        native.call("si_batch_rms_norm", h.data_ptr(), w["attn_norm_0"].data_ptr(), control.data_ptr(), normed.data_ptr(),
                    rows, hidden, cfg["epsilon"], stream)
        for layer, cache in enumerate(self.caches):
            def add_and_norm(update, norm):
                native.call("si_batch_residual_rms_norm", h.data_ptr(), update.data_ptr(), w[norm].data_ptr(),
                            control.data_ptr(), h.data_ptr(), normed.data_ptr(), rows, hidden, cfg["epsilon"], stream)

            qkv, query, mixed = project(f"qkv_weight_{layer}", normed), buffer(heads * d), buffer(heads * d)
            native.call("si_paged_rope_kv_append", C.byref(cache), native.F32, qkv.data_ptr(), qkv.shape[1],
                        starts.data_ptr(), lengths.data_ptr(), self.frequencies.data_ptr(), query.data_ptr(), heads * d,
                        rows, heads, cfg["rotary_size"], cfg["rope_scale"], stream)
            native.call("si_paged_attention", C.byref(cache), native.F32, query.data_ptr(), heads * d, starts.data_ptr(),
                        lengths.data_ptr(), mixed.data_ptr(), heads * d, rows, most, heads, d ** -0.5, 0,
                        self.workspace.data_ptr(), self.workspace.numel(), stream)
            add_and_norm(project(f"attn_output_weight_{layer}", mixed), f"ffn_norm_{layer}")
            gate_up, gated = project(f"ffn_up_weight_{layer}", normed), buffer(cfg["intermediate"])
            native.call("si_batch_swiglu", gate_up.data_ptr(), control.data_ptr(), gated.data_ptr(), rows,
                        cfg["intermediate"], stream)
            after = f"attn_norm_{layer + 1}" if layer + 1 < cfg["layers"] else "output_norm"
            add_and_norm(project(f"ffn_down_weight_{layer}", gated), after)

        def logits(last):
            x = normed[last].contiguous()
            y = torch.empty(len(last), cfg["vocab"], device="cuda")
            count = torch.tensor([0, len(last)], dtype=torch.int32, device="cuda")
            native.call("si_batch_shared_matvec", native.F16, w["token_embedding"].data_ptr(), x.data_ptr(),
                        count.data_ptr(), y.data_ptr(), len(last), cfg["vocab"], hidden, stream)
            return y

        return logits

    def _pick(self, logits, requests):
        vocab, stream, keep = self.cfg["vocab"], torch.cuda.current_stream().cuda_stream, []

        def dev(x, dtype):
            keep.append(torch.from_numpy(np.ascontiguousarray(x, dtype)).cuda())
            return keep[-1].data_ptr() if keep[-1].numel() else None

        history = [np.concatenate([r.prompt, np.asarray(r.tokens, np.int32)]) for r in requests]
        masks = [r.allowed for r in requests if r.allowed is not None]
        c = native.LogitControls()
        c.history, c.history_count = dev(np.concatenate(history), np.int32), sum(map(len, history))
        c.history_starts = dev(np.concatenate([[0], np.cumsum([len(h) for h in history])]), np.int32)
        c.repetition = dev([r.repetition for r in requests], np.float32)
        c.frequency = dev([r.frequency for r in requests], np.float32)
        c.presence = dev([r.presence for r in requests], np.float32)
        c.bias_tokens = dev([t for r in requests for t in r.biases], np.int32)
        c.bias_values = dev([v for r in requests for v in r.biases.values()], np.float32)
        c.bias_starts = dev(np.concatenate([[0], np.cumsum([len(r.biases) for r in requests])]), np.int32)
        c.bias_count = sum(len(r.biases) for r in requests)
        if masks:
            words = (vocab + 31) // 32
            bits = np.zeros((len(masks), words * 32), bool)
            bits[:, :vocab] = masks
            c.allowed = dev(np.packbits(bits, axis=1, bitorder="little").view(np.uint32), np.uint32)
            c.allowed_rows, c.allowed_stride = len(masks), words
            at = np.cumsum([r.allowed is not None for r in requests]) - 1
            c.allowed_index = dev([a if r.allowed is not None else -1 for a, r in zip(at, requests)], np.int32)
        picked = torch.empty(len(requests), dtype=torch.int32, device="cuda")
        native.call("si_process_logits", native.F32, logits.data_ptr(), vocab, C.byref(c), None, vocab, picked.data_ptr(),
                    len(requests), vocab, stream)
        return picked.cpu().numpy()

    def export(self, slot, layer, tokens):
        """The last tokens' keys and values of a slot as contiguous F16 rows, exactly as the cache holds them."""
        kv, d = self.cfg["kv_heads"], self.cfg["head_size"]
        starts = torch.zeros(self.slots + 1, dtype=torch.int32)
        starts[slot + 1:] = tokens
        lengths = torch.tensor([r.held if r else 0 for r in self.active], dtype=torch.int32, device="cuda")
        starts = starts.cuda()
        k, v = (torch.zeros(tokens, kv * d, dtype=torch.float16, device="cuda") for _ in range(2))
        native.call("si_paged_kv_gather", C.byref(self.caches[layer]), native.F16, starts.data_ptr(), lengths.data_ptr(),
                    k.data_ptr(), v.data_ptr(), tokens, torch.cuda.current_stream().cuda_stream)
        torch.cuda.current_stream().synchronize()
        return k, v


def random_model(cfg, seed):
    weights = dict(phi4.synthetic_weights(cfg, seed))
    for name in native.decoder_slot_names(cfg["layers"]):
        if name not in weights:
            weights[name] = np.ones(cfg["hidden"], np.float32)
    return weights


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--requests", type=int, default=6)
    p.add_argument("--slots", type=int, default=4)
    p.add_argument("--tokens", type=int, default=24)
    args = p.parse_args()
    cfg = dict(phi4.TINY, context=1024, weight_type=native.F16, embedding_type=native.F16)
    server = PagedServer(cfg, random_model(cfg, 1), args.slots, pages=args.slots * 16, chunk=256)
    requests = []
    for i in range(args.requests):
        even = np.arange(cfg["vocab"]) % 2 == 0
        requests.append(Request(phi4.random_prompt(i, 40 + 170 * i % 700, cfg["vocab"]), args.tokens, repetition=1.3,
                                frequency=0.05, biases={7: -1.0}, allowed=even if i % 2 else None))
        server.submit(requests[-1])
    server.run()
    for i, r in enumerate(requests):
        print(f"request {i} ({len(r.prompt)} prompt tokens): {r.tokens}")


if __name__ == "__main__":
    main()
