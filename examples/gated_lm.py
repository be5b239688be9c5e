"""A small language model around the gated linear recurrence, with the operators as a program uses them:

    tokens -> embedding_fwd (scaled) -> [ RMSNorm -> projection x | f | z -> gated_scan -> projection ] x layers
           -> RMSNorm -> tied head -> token_logprobs

`train_step` is one manual forward, backward and AdamW step on next-token prediction with an entropy bonus, `score` gives the log
probability of every token of a text with its alternatives, `generate` decodes token by token from a carried state.  The dense
products are torch.matmul; everything else is this library.

    python examples/gated_lm.py          # trains a little model on a repeating text and continues it
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import mamba_rs_b200 as mb  # noqa: E402


class GatedLM:
    """Parameters live in one flat f32 arena with a copy in the compute dtype and a gradient arena beside it."""

    def __init__(self, vocab, d_model, d_inner, layers, device="cuda", dtype=torch.bfloat16, seed=0):
        self.vocab, self.d, self.D, self.layers, self.dtype = vocab, d_model, d_inner, layers, dtype
        self.scale = math.sqrt(d_model)
        shapes = [("table", (vocab, d_model)), ("norm_f", (d_model,))]
        for i in range(layers):
            shapes += [(f"norm{i}", (d_model,)), (f"in{i}", (d_model, 3 * d_inner)), (f"out{i}", (d_inner, d_model))]
        n = sum(-(-math.prod(s) // 64) * 64 for _, s in shapes)
        self.master, self.grad, self.m, self.v = (torch.zeros(n, device=device) for _ in range(4))
        self.lp = self.master if dtype == torch.float32 else torch.empty(n, device=device, dtype=dtype)
        self.p, self.w, self.g, at = {}, {}, {}, 0
        for name, s in shapes:
            size = math.prod(s)
            self.p[name], self.w[name], self.g[name] = (a[at:at + size].view(s) for a in (self.master, self.lp, self.grad))
            at += -(-size // 64) * 64
        g = torch.Generator(self.master.device).manual_seed(seed)
        for name, t in self.p.items():
            if name.startswith("norm"):
                t.fill_(1.0)
            else:
                t.normal_(0.0, 1.0 / self.scale if name == "table" else t.shape[0] ** -0.5, generator=g)
        if self.lp is not self.master:
            self.lp.copy_(self.master)
        self.steps, self.bias = 0, torch.ones(2, device=device)

    def state(self, batch):
        """Recurrent state of every layer before the first token."""
        return torch.zeros(self.layers, batch, self.D, device=self.master.device)

    # ---- whole texts ----
    def _hidden(self, ids, state, keep):
        """Normalised rows [B*T, d] behind the last layer; `state` is carried on; keep: a list that gets what the backward needs."""
        B, T = ids.shape
        res, branch = mb.embedding_fwd(self.w["table"], ids, scale=self.scale), None
        for i in range(self.layers):
            n, rms = mb.residual_rmsnorm_fwd(res, branch, self.p[f"norm{i}"], out_dtype=self.dtype)
            proj = (n @ self.w[f"in{i}"]).view(B, T, 3 * self.D)
            x, f, z = proj.split(self.D, 2)
            blocks = torch.empty(mb.gated_scan_states(B, T, self.D), device=res.device) if keep is not None else None
            y = mb.gated_scan_fwd(x, f, z, h0=state[i], h_last=state[i], chunk_states=blocks)
            if keep is not None:
                keep.append((res.clone(), n, rms, proj, blocks, y))
            branch = y.view(B * T, self.D) @ self.w[f"out{i}"]
        n, rms = mb.residual_rmsnorm_fwd(res, branch, self.p["norm_f"], out_dtype=self.dtype)
        if keep is not None:
            keep.append((res, n, rms))
        return n

    def score(self, ids, state=None, top=0, temperature=1.0, rows=4096):
        """ids [B,T] int32: of each token behind the first its log probability, entropy and alternatives, [B, T-1, ...]; the
        logits of at most `rows` positions exist at a time."""
        B, T = ids.shape
        hidden = self._hidden(ids[:, :-1].contiguous(), self.state(B) if state is None else state, None)
        targets = ids[:, 1:].reshape(-1).contiguous()
        parts = [mb.token_logprobs(hidden[r:r + rows] @ self.w["table"].t(), targets[r:r + rows], top=top, temperature=temperature)
                 for r in range(0, hidden.shape[0], rows)]
        return {k: torch.cat([p[k] for p in parts]).view(B, T - 1, *parts[0][k].shape[1:]) for k in parts[0] if k != "lse"}

    def gradients(self, ids, entropy_bonus=0.0):
        """Accumulates the gradient of -mean(log p(next token)) - entropy_bonus * mean(entropy); returns that loss."""
        B, T = ids.shape[0], ids.shape[1] - 1
        keep, inputs = [], ids[:, :-1].contiguous()
        hidden = self._hidden(inputs, self.state(B), keep)
        targets = ids[:, 1:].reshape(-1).contiguous()
        logits = hidden @ self.w["table"].t()
        r = mb.token_logprobs(logits, targets)
        n = B * T
        loss = -(r["logprob"].sum() + entropy_bonus * r["entropy"].sum()) / n
        row = torch.full((n,), -1.0 / n, device=logits.device)
        # the gradient takes the logits' place
        d = mb.token_logprobs_bwd(logits, targets, r["lse"], r["entropy"], row, row * entropy_bonus, dlogits=logits)
        self._add(self.g["table"], d, hidden)
        d_n = d @ self.w["table"]
        res, _, rms = keep.pop()
        d_res = torch.zeros_like(res)
        mb.residual_rmsnorm_bwd(d_n, res, self.p["norm_f"], rms, d_res, self.g["norm_f"])
        for i in range(self.layers - 1, -1, -1):
            res, norm, rms, proj, blocks, y = keep.pop()
            d_branch = d_res.to(self.dtype)
            self._add(self.g[f"out{i}"], y.view(n, self.D), d_branch)
            dy = (d_branch @ self.w[f"out{i}"].t()).view(B, T, self.D)
            d_proj = torch.empty_like(proj)
            x, f, z = proj.split(self.D, 2)
            dx, df, dz = d_proj.split(self.D, 2)
            mb.gated_scan_bwd(x, f, dy, blocks, z, d_x=dx, d_f=df, d_z=dz)
            d_proj = d_proj.view(n, 3 * self.D)
            self._add(self.g[f"in{i}"], norm, d_proj)
            mb.residual_rmsnorm_bwd(d_proj @ self.w[f"in{i}"].t(), res, self.p[f"norm{i}"], rms, d_res, self.g[f"norm{i}"])
        mb.embedding_bwd(inputs, d_res, d_table=self.g["table"], scale=self.scale)
        return loss

    @staticmethod
    def _add(g, a, b):
        """g (f32) += a^T b."""
        if a.dtype == torch.float32:
            g.addmm_(a.t(), b)
        else:
            torch.addmm(g, a.t(), b, out_dtype=torch.float32, out=g)

    def train_step(self, ids, lr=3e-3, entropy_bonus=0.0, betas=(0.9, 0.95)):
        """One step on ids [B, T+1] int32; returns the loss (a device scalar)."""
        loss = self.gradients(ids, entropy_bonus)
        self.steps += 1
        for i, b in enumerate(betas):
            self.bias[i:i + 1].fill_(1.0 / (1.0 - b ** self.steps))
        mb.adamw_step(self.master, self.grad, self.m, self.v, self.bias, lr=lr, beta1=betas[0], beta2=betas[1],
                      param_lp=None if self.lp is self.master else self.lp)
        self.grad.zero_()
        return loss

    # ---- token by token ----
    def step(self, ids, state, top=1):
        """One token per sequence: ids [B] int32, the state is updated in place; token_logprobs of what comes next."""
        res, branch = mb.embedding_fwd(self.w["table"], ids, scale=self.scale), None
        for i in range(self.layers):
            n, _ = mb.residual_rmsnorm_fwd(res, branch, self.p[f"norm{i}"], out_dtype=self.dtype)
            x, f, z = (n @ self.w[f"in{i}"]).split(self.D, 1)
            branch = mb.gated_scan_step(x, f, state[i], z) @ self.w[f"out{i}"]
        n, _ = mb.residual_rmsnorm_fwd(res, branch, self.p["norm_f"], out_dtype=self.dtype)
        return mb.token_logprobs(n @ self.w["table"].t(), top=top)

    def generate(self, prompt, n, top=1):
        """n tokens behind prompt [B,T] int32, the most likely one each time: tokens [B,n], their log probabilities [B,n], and the
        alternatives [B,n,top] with theirs."""
        B, T = prompt.shape
        state = self.state(B)
        hidden = self._hidden(prompt.contiguous(), state, None).view(B, T, self.d)[:, -1]
        r, out = mb.token_logprobs(hidden @ self.w["table"].t(), top=top), []
        for i in range(n):
            out.append((r["top_ids"], r["top_logprobs"]))
            if i + 1 < n:
                r = self.step(r["top_ids"][:, 0].contiguous(), state, top)
        ids, lp = (torch.stack(t, 1) for t in zip(*out))
        return ids[..., 0], lp[..., 0], ids, lp


def main():
    text = torch.tensor([ord(c) for c in "the state forgets, the state keeps. " * 24], dtype=torch.int32, device="cuda")
    lm = GatedLM(vocab=128, d_model=128, d_inner=256, layers=2)
    windows = torch.stack([text[i:i + 257] for i in range(0, 36 * 8, 36 + 7)])
    for i in range(200):
        loss = lm.train_step(windows, entropy_bonus=1e-3)
        if i % 50 == 0 or i == 199:
            print(f"step {i}: loss {float(loss):.3f}")
    prompt = text[None, :40].contiguous()
    ids, lp, alternatives, _ = lm.generate(prompt, 36, top=3)
    print(repr("".join(map(chr, ids[0].tolist()))), f"log p {float(lp.sum()):.2f}")
    print("score of the text:", f"{float(lm.score(text[None, :257])['logprob'].mean()):.3f} nats a token")


if __name__ == "__main__":
    main()
