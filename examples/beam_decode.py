"""Beam search over encoder features with the paged cache and the token scores.

    python examples/beam_decode.py [--clips 4] [--beams 5] [--steps 40]

A Whisper-shaped encoder and text decoder with random weights (there is no
checkpoint here, so the tokens mean nothing): the encoder's frames are written once
into a paged cache for cross attention, where the beams of a clip are one group of
queries over its keys; self attention has a paged cache of its own, whose beams are
reordered by kv_fork after every step; token_logprobs gives each step's candidates.
"""
import argparse
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "whisper-xdna_b200"))
from wxb200 import _lib as L  # noqa: E402
from wxb200 import ops  # noqa: E402
from wxb200.encoder import Encoder, synthetic_weights  # noqa: E402
from wxb200.kvcache import PagedKVCache  # noqa: E402


def decoder_weights(d=384, ffn=1536, n_layer=2, vocab=2003, n_text=64, seed=2):
    """Random weights: bf16 matrices in the torch Linear layout (out, in), fp32 biases
    and LayerNorm parameters."""
    g = torch.Generator().manual_seed(seed)
    mat = lambda *s: (torch.randn(*s, generator=g) * s[-1] ** -0.5).to(torch.bfloat16).cuda()  # noqa: E731
    vec = lambda n: (torch.randn(n, generator=g) * 0.02).cuda()  # noqa: E731
    ln = lambda: (1 + vec(d), vec(d))  # noqa: E731
    layers = [{"ln1": ln(), "qkv": (mat(3 * d, d), vec(3 * d)), "out": (mat(d, d), vec(d)),
               "ln2": ln(), "q2": (mat(d, d), vec(d)), "kv2": (mat(2 * d, d), vec(2 * d)),
               "out2": (mat(d, d), vec(d)), "ln3": ln(), "fc1": (mat(ffn, d), vec(ffn)),
               "fc2": (mat(d, ffn), vec(d))} for _ in range(n_layer)]
    return {"layers": layers, "embed": mat(vocab, d) * 2, "pos": mat(n_text, d).float(),
            "ln": ln()}


class BeamDecoder:
    """A text decoder's step for clips x beams sequences on the framework's operators."""

    def __init__(self, W, features, beams, page_size=16):
        """features: (clips, frames, d) fp32 from the encoder."""
        self.W, self.beams = W, beams
        clips, frames, d = features.shape
        self.clips, self.d, self.heads = clips, d, d // 64
        n_layer, n_text = len(W["layers"]), W["pos"].shape[0]
        n = clips * beams
        width = -(-n_text // page_size)
        self.cache = PagedKVCache(n_layer, n * width + n, page_size, self.heads, 64, n, n_text)
        # the frames' keys and values, once a layer: one sequence a clip
        per_clip = -(-frames // 64)
        self.frames = PagedKVCache(n_layer, clips * per_clip, 64, self.heads, 64, clips, frames)
        all_frames = torch.full((clips,), frames, dtype=torch.int32, device="cuda")
        self.frames.step(grow=all_frames)
        x = features.reshape(clips * frames, d).to(torch.bfloat16)
        for i, w in enumerate(W["layers"]):
            kv = ops.gemm(x, *w["kv2"], epilogue=L.WX_EPI_BF16).view(clips, frames, 2,
                                                                    self.heads, 64)
            self.frames.append(i, kv[:, :, 0], kv[:, :, 1])

    def _norm(self, x, ln):
        return ops.layer_norm_rows(x, *ln, mode=L.WX_LN_FP32, out_dtype=torch.bfloat16)

    def step(self, tokens, position, parents=None):
        """Logits (clips * beams, vocab) fp32 after `tokens` (int64) at `position`, the
        sequences going on as `parents` were."""
        n, d, heads = tokens.shape[0], self.d, self.heads
        self.cache.step(parents, torch.ones(n, dtype=torch.int32, device="cuda"))
        x = self.W["embed"][tokens].float() + self.W["pos"][position]
        for i, w in enumerate(self.W["layers"]):
            qkv = ops.gemm(self._norm(x, w["ln1"]), *w["qkv"], epilogue=L.WX_EPI_BF16)
            q, k, v = qkv.view(n, 3, heads, 64).unbind(1)
            self.cache.append(i, k, v)
            o = self.cache.attend(i, q.contiguous())
            x = ops.gemm(o.view(n, d), *w["out"], residual=x)
            q = ops.gemm(self._norm(x, w["ln2"]), *w["q2"], epilogue=L.WX_EPI_BF16)
            # a clip's beams are one group of queries over its frames
            o = self.frames.attend(i, q.view(self.clips, self.beams, heads, 64).transpose(1, 2))
            x = ops.gemm(o.transpose(1, 2).reshape(n, d), *w["out2"], residual=x)
            h = ops.gemm(self._norm(x, w["ln3"]), *w["fc1"], epilogue=L.WX_EPI_BF16_GELU_ERF)
            x = ops.gemm(h, *w["fc2"], residual=x)
        vocab = self.W["embed"].shape[0]
        logits = torch.empty(n, -(-vocab // 4) * 4, device="cuda")[:, :vocab]   # aligned rows
        return ops.gemm(self._norm(x, self.W["ln"]), self.W["embed"], out=logits)


def beam_search(decoder, start, steps, compact_at=None):
    """The best `beams` hypotheses of each clip after `steps` tokens: (tokens
    (clips, beams, steps) int64, summed log probabilities (clips, beams))."""
    clips, beams = decoder.clips, decoder.beams
    n = clips * beams
    tokens = torch.full((n,), start, dtype=torch.int64, device="cuda")
    none = torch.full((n,), -1, dtype=torch.int64, device="cuda")
    total = torch.full((clips, beams), -float("inf"), device="cuda")
    total[:, 0] = 0                                # all beams start alike: one counts
    history = torch.empty(n, 0, dtype=torch.int64, device="cuda")
    first = torch.arange(clips, device="cuda")[:, None] * beams
    parents = None
    for t in range(steps):
        logits = decoder.step(tokens, t, parents)
        _, _, value, index = ops.token_logprobs(logits, none, top_k=beams)
        total, pick = (total[:, :, None] + value.view(clips, beams, beams)).flatten(1).topk(
            beams, dim=1)
        rows = (first + pick // beams).flatten()   # which beam each goes on from
        parents = rows.to(torch.int32)
        tokens = index.view(clips, beams * beams).gather(1, pick).flatten().long()
        history = torch.cat([history[rows], tokens[:, None]], dim=1)
        if t == compact_at:
            decoder.cache.compact()
    return history.view(clips, beams, steps), total


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--clips", type=int, default=4)
    ap.add_argument("--beams", type=int, default=5)
    ap.add_argument("--steps", type=int, default=40)
    a = ap.parse_args()
    W = decoder_weights(n_text=a.steps + 1)
    enc = Encoder(synthetic_weights(n_mels=80, d=384, ffn=1536, n_layer=2, n_ctx=1500),
                  max_batch=a.clips)
    gen = torch.Generator(device="cuda").manual_seed(0)
    mel = torch.rand(a.clips, 80, 3000, device="cuda", generator=gen) * 2 - 0.8
    features = enc.forward(mel)
    tokens, total = beam_search(BeamDecoder(W, features, a.beams), start=1, steps=a.steps)
    for c in range(a.clips):
        mean = total[c, 0].item() / a.steps
        print(f"clip {c}: mean log probability {mean:.3f}, tokens {tokens[c, 0, :12].tolist()} ...")


if __name__ == "__main__":
    main()
