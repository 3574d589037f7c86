"""Attention of a served model end to end on packed E8 weights and an E8 key/value cache.

    python examples/cached_attention.py

One layer: query, key, value and output projections are QAT layers exported
to packed codes (PackedLinear); queries and keys are normalized by head and
rotated (qk_norm_rope); keys and values go into a paged cache as E8 points
(kv_write); attention runs over the cache (kv_attention).  A prompt is taken
in two chunks, tokens are decoded one at a time, and a tree of drafted tokens
is scored in one call.  The result of each is compared with attention in fp32
over the cache's rows read back (kv_read).
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import coset_amd as ca  # noqa: E402

WIDTH, HEADS, KV_HEADS, DIM, PAGE = 768, 12, 4, 64, 32


def packed(fin, fout):
    """A QAT layer's packed form (its weights as trained, here as initialized)."""
    layer = ca.create_e8_hnlq_linear(fin, fout, q=4, M=2, Delta0=1.5, weight_clip_value=10.0)
    with torch.no_grad():
        layer.weight.normal_(0.0, 0.5)
    layer(torch.randn(8, fin, device="cuda")).sum().backward()   # one step: the scale's running statistics
    with torch.no_grad():
        st = ca.packed_state(layer)
    return ca.PackedLinear(st["tensors"], st["metadata"])


class CachedAttention:
    def __init__(self, seqs, max_tokens, bits):
        self.qkv = packed(WIDTH, (HEADS + 2 * KV_HEADS) * DIM)
        self.proj = packed(HEADS * DIM, WIDTH)
        self.q_norm = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
        self.k_norm = torch.ones(DIM, dtype=torch.bfloat16, device="cuda")
        self.table = ca.rope_table(max_tokens, DIM)
        pages = -(-max_tokens // PAGE)
        self.cache = ca.E8KVCache.empty(seqs * pages, PAGE, KV_HEADS, DIM, bits)
        # a sequence's pages; a server would hand them out as sequences grow
        self.pages = torch.randperm(seqs * pages, device="cuda").view(seqs, pages).int()
        self.lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")

    def slots(self, seq, place):
        return self.pages[seq, place // PAGE].long() * PAGE + place % PAGE

    def __call__(self, x, depth=None, tree_mask=None):
        """x [seqs, new, WIDTH], tokens that follow the cached ones.  depth [new]: how far behind the cached tokens
        each stands (its own number, or a drafted token's depth in its tree)."""
        seqs, new, _ = x.shape
        n = seqs * new
        qkv = self.qkv(x.reshape(n, WIDTH)).to(torch.bfloat16)
        q, k, v = qkv.split([HEADS * DIM, KV_HEADS * DIM, KV_HEADS * DIM], dim=1)
        seq = torch.arange(seqs, device="cuda").repeat_interleave(new)
        own = torch.arange(new, device="cuda").repeat(seqs)
        before = self.lengths[seq].long()
        positions = before + (own if depth is None else depth.repeat(seqs))
        q, k = ca.qk_norm_rope(q.view(n, HEADS, DIM), k.view(n, KV_HEADS, DIM), self.table, positions, self.q_norm,
                               self.k_norm)
        ca.kv_write(self.cache, k, v.view(n, KV_HEADS, DIM), self.slots(seq, before + own))
        self.lengths += new
        mask = None if tree_mask is None else tree_mask.repeat(seqs, 1)
        out = ca.kv_attention(q, self.cache, self.pages, self.lengths, tree_mask=mask)
        self.last = q, out, mask
        return self.proj(out.reshape(n, HEADS * DIM)).view(seqs, new, WIDTH)

    def dense(self, new):
        """The last call's attention in fp32 over the rows read back."""
        q, out, mask = self.last
        worst = 0.0
        for b in range(self.pages.shape[0]):
            length = int(self.lengths[b])
            place = torch.arange(length, device="cuda")
            k, v = ca.kv_read(self.cache, self.slots(torch.full_like(place, b), place), torch.float32)
            rows = q[b * new:(b + 1) * new].float()
            draft = place - (length - new)
            if mask is None:
                seen = draft <= torch.arange(new, device="cuda")[:, None]
            else:
                seen = (draft < 0) | ((mask[b * new:(b + 1) * new] >> draft.clamp(min=0)) & 1 == 1)
            for h in range(HEADS):
                s = rows[:, h] @ k[:, h // (HEADS // KV_HEADS)].t().contiguous() * DIM ** -0.5
                want = torch.softmax(s.masked_fill(~seen, float("-inf")), dim=1) @ v[:, h // (HEADS // KV_HEADS)]
                off = float((out[b * new:(b + 1) * new, h].float() - want).abs().max() / want.abs().max())
                if not off < 1.0:
                    raise RuntimeError(f"head {h} of sequence {b} is not the attention over its cache: {off}")
                worst = max(worst, off)
        return worst


def main(bits=4):
    torch.manual_seed(0)
    seqs = 3
    layer = CachedAttention(seqs, 1024, bits)
    worst = 0.0
    for new in (300, 77):                     # a prompt in two chunks
        layer(torch.randn(seqs, new, WIDTH, device="cuda").bfloat16())
        worst = max(worst, layer.dense(new))
    for _ in range(5):                        # tokens one at a time
        layer(torch.randn(seqs, 1, WIDTH, device="cuda").bfloat16())
        worst = max(worst, layer.dense(1))
    parents = [-1, 0, 0, 1, 1, 2, -1, 6]      # a tree of drafted tokens
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    mask = ca.draft_tree_mask(torch.tensor(parents, device="cuda"))
    layer(torch.randn(seqs, len(parents), WIDTH, device="cuda").bfloat16(), torch.tensor(depth, device="cuda"), mask)
    worst = max(worst, layer.dense(len(parents)))
    layer.lengths -= len(parents)             # the path that was accepted would be written again, behind the context
    print(f"{bits}-bit cache of {layer.cache.nbytes() / 2 ** 20:.1f} MiB, {int(layer.lengths[0])} tokens in each of "
          f"{seqs} sequences: largest difference from dense attention over the cached values {worst:.2e}")
    return worst


if __name__ == "__main__":
    for b in (4, 8):
        main(b)
