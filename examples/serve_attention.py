"""One decoder layer's attention block as a server runs it: the MXFP4 QKV
Linear, norms, rotation and the append to the 4-bit cache, attention over the
cache, and the output Linear on the attention's MXINT8 copy.

    python examples/serve_attention.py

Prompts of several requests go through together, then tokens one by one; the
requests share one pool of cache pages.  The sizes are SmolVLA's language
model (960 wide, 15 query heads over 5 key/value heads of 64).  Weights and
inputs are random.
"""
from __future__ import annotations

import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from hotarubi_b200 import capi, workloads  # noqa: E402


class AttentionBlock:
    """The block's weights, the page pool and the requests' state."""

    def __init__(self, lib: capi.Library, *, requests: int, max_kv: int, hidden=960, heads=15,
                 kv_heads=5, hd=64, page=16, seed=0):
        self.lib, self.hidden, self.heads, self.kv_heads, self.hd = lib, hidden, heads, kv_heads, hd
        self.requests, self.page, self.max_kv = requests, page, max_kv
        dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
        self.qkv_n = (heads + 2 * kv_heads) * hd
        self.w_qkv = [dev(x) for x in workloads.mxfp4_weights(seed, self.qkv_n, hidden)]
        self.w_out = [dev(x) for x in workloads.mxfp4_weights(seed + 1, hidden, heads * hd)]
        self.q_norm, self.k_norm = (torch.ones(hd, device="cuda") for _ in range(2))
        self.rope = dev(capi.rope_table(max_kv, hd))
        i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device="cuda")  # noqa: E731
        self.table_ld = -(-max_kv // page)
        pages = requests * self.table_ld
        self.cache_bytes = torch.zeros(pages * kv_heads * capi.kv_record_bytes(page, hd),
                                       dtype=torch.uint8, device="cuda")
        self.cache = capi.kv_cache(self.cache_bytes, pages, page, kv_heads, hd)
        self.free = torch.randperm(pages, device="cuda").int()
        self.head, self.next_head = i32(1), i32(1)
        self.table = torch.full((requests, self.table_ld), -1, dtype=torch.int32, device="cuda")
        self.cached, self.kv_len, self.q_start = i32(requests), i32(requests), i32(requests + 1)
        self.lengths = [0] * requests  # the host's own count, for the call's bounds
        torch.cuda.synchronize()

    def step(self, x: torch.Tensor, fresh: list[int]) -> torch.Tensor:
        """x: FP32 [sum(fresh)][hidden], request by request; the block's output
        for these tokens.  Everything runs on the library's stream."""
        lib, n = self.lib, x.shape[0]
        assert n == sum(fresh) and len(fresh) == self.requests
        width = self.heads * self.hd
        new = torch.tensor(fresh, dtype=torch.int32, device="cuda")
        slots, pos = (torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(2))
        qkv = torch.empty(n, self.qkv_n, device="cuda")
        q = torch.empty(n, width, dtype=torch.bfloat16, device="cuda")
        codes = torch.empty(n, width, dtype=torch.int8, device="cuda")
        scales = torch.empty(n, width // 32, dtype=torch.uint8, device="cuda")
        y = torch.empty(n, self.hidden, device="cuda")
        self.lengths = [a + b for a, b in zip(self.lengths, fresh)]
        torch.cuda.synchronize()  # torch's copies run on another stream
        lib.block_tables(capi.blocks_desc(
            self.requests, self.page, cached=self.cached, fresh=new, free_pages=self.free,
            nfree=self.free.numel(), head_in=self.head, head_out=self.next_head, table=self.table,
            table_ld=self.table_ld, q_start=self.q_start, kv_len=self.kv_len, slots=slots, pos=pos,
            max_tokens=n))
        lib.dense(capi.Library.desc(capi.WFMT_MXFP4, n, self.qkv_n, self.hidden, a=x, w=self.w_qkv[0],
                                    wscale=self.w_qkv[1], c=qkv, mode=capi.MODE_FAST))
        lib.qkv_append(capi.qkv_desc(
            self.cache, n, self.heads, q=qkv, k=qkv[:, width:], v=qkv[:, width + self.kv_heads * self.hd:],
            ldq=self.qkv_n, ldk=self.qkv_n, ldv=self.qkv_n, q_norm=self.q_norm, k_norm=self.k_norm,
            rope=self.rope, max_pos=self.max_kv, rot=self.hd, pos=pos, slots=slots, q_out=q))
        lib.attention(capi.attn_desc(
            self.cache, self.requests, self.heads, q=q, q_start=self.q_start, total_q=n,
            max_q=max(fresh), kv_len=self.kv_len, max_kv=max(self.lengths),
            total_kv=sum(self.lengths), table=self.table, table_ld=self.table_ld,
            scale=self.hd ** -0.5, oq=codes, oscale=scales))
        lib.dense(capi.Library.desc(capi.WFMT_MXFP4, n, self.hidden, width, aq=codes, ascale=scales,
                                    w=self.w_out[0], wscale=self.w_out[1], c=y))
        lib.sync()
        self.cached.copy_(self.kv_len)
        self.head, self.next_head = self.next_head, self.head
        return y


def main() -> None:
    lib = capi.Library(0)
    prompts = [141, 37, 90]
    block = AttentionBlock(lib, requests=len(prompts), max_kv=256)
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(sum(prompts), block.hidden, device="cuda", generator=gen)
    y = block.step(x, prompts)
    print(f"prompts {prompts}: output {tuple(y.shape)}, rms {y.square().mean().sqrt().item():.4f}")
    for _ in range(20):
        x = torch.randn(len(prompts), block.hidden, device="cuda", generator=gen)
        y = block.step(x, [1] * len(prompts))
    print(f"after 20 tokens each: lengths {block.lengths}, rms {y.square().mean().sqrt().item():.4f}, "
          f"{lib.launches()} kernel launches")
    lib.close()


if __name__ == "__main__":
    main()
