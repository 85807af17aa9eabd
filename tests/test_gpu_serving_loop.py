"""Prompt, single tokens, verify blocks, branches, trimming and compaction as a serving loop chains them, over one paged
cache, against the 64-bit statement that keeps every request's keys and values as plain lists."""
import pytest
import torch

from oracle import attention as oattn

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn
HKV, D, PAGE = 2, 128, 16
WIDE = 18 * HKV * D


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Server:
    """A pool, its caches, and for every row the K/V bytes it should see (position -> bytes), copied from the cache when
    written."""

    def __init__(self, window, sinks, pages_n=60, rows=6):
        from muse_spark_open_b200 import pages
        self.pool = pages.prepare(pages_n, PAGE, rows, 40)
        self.kc, self.vc = (torch.full((pages_n, PAGE, HKV, D), 0x7F, dtype=torch.uint8, device="cuda").view(FP8) for _ in range(2))
        self.cfg = {"num_q_heads": 8 * HKV, "num_kv_heads": HKV, "head_dim": D, "page_size": PAGE, "window": window, "sinks": sinks, "rope_theta": 1e4,
                    "qk_scale_factor": oattn.QK_SCALE_FACTOR, "sm_scale": D ** -0.5}
        self.scale = torch.tensor(3.0 / 448, device="cuda")
        self.gen = torch.Generator().manual_seed(window + sinks)
        self.seen = [[] for _ in range(rows)]  # per row: (k, v) uint8 [HKV, D] per position

    def step(self, rows, counts, how):
        """New tokens for `rows`; checks the outputs and remembers what was written."""
        from muse_spark_open_b200 import abi, attention, pages
        cu = [0] + torch.tensor(counts).cumsum(0).tolist()
        qkv = torch.randn((cu[-1], WIDE), generator=self.gen)
        qkv[:, :9 * HKV * D] *= 2
        qkv = qkv.to(torch.bfloat16)
        r = i32(rows)
        if how == "prompt":
            loc = pages.extend(self.pool, r, cu_seqlens=i32(cu), tokens=cu[-1])
        else:
            loc = pages.extend(self.pool, r, counts[0])
        table, seq = self.pool["page_table"][r.long()].contiguous(), self.pool["seq_lens"][r.long()].contiguous()
        data = {"qkv": qkv.cuda(), "seq_lens": seq, "page_table": table, "k_cache": self.kc, "v_cache": self.vc, "k_scale": self.scale, "v_scale": self.scale,
                "config": dict(self.cfg, batch=len(rows), q_len=counts[0])}
        if how == "prompt":
            out = attention.prompt_fn(dict(data, cu_seqlens_q=i32(cu)))
        else:
            out = attention.kernel_fn(dict(data, cache_loc=loc)).view(cu[-1], -1)
        torch.cuda.synchronize()
        abi.status_for("cuda").raise_if_set("serving loop")
        k_new, v_new = (c.view(torch.uint8).view(-1, HKV, D)[loc].cpu() for c in (self.kc, self.vc))
        # the statement: a cache of its own, one row after another
        ctx = [len(self.seen[x]) for x in rows]
        most = max(c + n for c, n in zip(ctx, counts))
        cols = (most + PAGE - 1) // PAGE
        kc, vc = (torch.zeros(len(rows) * cols, PAGE, HKV, D, dtype=torch.uint8) for _ in range(2))
        for j, x in enumerate(rows):
            if self.seen[x]:
                kc.view(len(rows), -1, HKV, D)[j, :ctx[j]] = torch.stack([a for a, _ in self.seen[x]])
                vc.view(len(rows), -1, HKV, D)[j, :ctx[j]] = torch.stack([b for _, b in self.seen[x]])
        ref_data = {"qkv": qkv, "k_cache": kc.view(FP8), "v_cache": vc.view(FP8), "k_scale": self.scale.cpu(), "v_scale": self.scale.cpu(),
                    "page_table": torch.arange(len(rows) * cols, dtype=torch.int32).view(len(rows), cols), "seq_lens": torch.tensor(ctx, dtype=torch.int32),
                    "cu_seqlens_q": torch.tensor(cu, dtype=torch.int32), "config": data["config"]}
        ref, rk, _ = oattn.ref_stream(ref_data, new_kv=(k_new.view(FP8), v_new.view(FP8)))
        got = out.cpu().double()
        assert torch.isfinite(got).all()
        # decode's queries are two E4M3 terms: the bounds of tests/test_gpu_sinks.py
        assert float((got - ref).norm() / ref.norm()) < 6e-3, (how, rows, counts)
        for j, x in enumerate(rows):
            self.seen[x] += [(k_new[t], v_new[t]) for t in range(cu[j], cu[j + 1])]
        self.pool["seq_lens"][r.long()] += i32(counts)

    def fork(self, parents, children):
        from muse_spark_open_b200 import pages
        pages.fork(self.pool, i32(parents), i32(children), [self.kc, self.vc])
        for p, c in zip(parents, children):
            self.seen[c] = list(self.seen[p])

    def free(self, rows):
        from muse_spark_open_b200 import pages
        pages.free(self.pool, i32(rows))
        for x in rows:
            self.seen[x] = []

    def check_pages(self):
        """refs count the table's entries; every position a later token sees is where the table says."""
        torch.cuda.synchronize()
        table, seq, refs = (self.pool[n].cpu() for n in ("page_table", "seq_lens", "refs"))
        count = torch.zeros_like(refs)
        for x in table[table >= 0].tolist():
            count[x] += 1
        assert torch.equal(count, refs)
        w, sinks = self.cfg["window"], self.cfg["sinks"]
        k = self.kc.view(torch.uint8).cpu()
        for row, seen in enumerate(self.seen):
            assert int(seq[row]) == len(seen)
            for s, (a, _) in enumerate(seen):
                if not w or s > len(seen) - w or s < sinks:
                    assert torch.equal(k[int(table[row, s // PAGE]), s % PAGE], a), (row, s)
        return int((refs > 0).sum())


@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 4), (33, 20)])
def test_serving_loop(window, sinks):
    from muse_spark_open_b200 import pages
    s = Server(window, sinks)
    s.step([0, 2, 1], [37, 100, 1], "prompt")
    s.step([2, 0, 1], [1, 1, 1], "tokens")
    s.fork([2, 0], [4, 3])
    s.step([0, 1, 2, 3, 4], [1] * 5, "tokens")
    s.step([4, 3], [8, 8], "verify")
    pages.trim(s.pool, i32([0, 1, 2, 3, 4]), window, sinks)
    s.check_pages()
    s.step([3, 0], [5, 70], "prompt")
    s.free([2])
    pages.trim(s.pool, i32([0, 1, 3, 4]), window, sinks)
    used = s.check_pages()
    assert pages.compact(s.pool, [s.kc, s.vc]).tolist()[0] == used
    assert s.check_pages() == used and not s.pool["refs"][used:].any()
    s.step([0, 1, 3, 4], [3] * 4, "blocks of three")
    s.fork([0, 0], [2, 5])
    s.step([0, 2, 5], [8, 8, 8], "verify")
    s.step([1, 2, 3, 4, 5], [1] * 5, "tokens")
    s.check_pages()
    s.free([0, 1, 2, 3, 4, 5])
    assert s.check_pages() == 0
