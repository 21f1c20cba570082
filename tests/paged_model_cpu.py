"""The model's paged path on the CPU, for tests of its host logic: the kernels' calls as plain torch on pools of bf16 rows."""

import torch

from exp3_b200 import model as model_module
from exp3_b200.model import AttentionSettings, Qwen2Config, Qwen2Model

CFG = Qwen2Config(vocab_size=64, hidden_size=256, intermediate_size=256, num_hidden_layers=2, num_attention_heads=12,
                  num_key_value_heads=2)


def _rows(page_table, pool, b, positions):
    size = pool.shape[2]
    return page_table[b, positions // size].long(), positions % size


class PlainPaged:
    """What model.py uses of exp3_b200.paged."""

    def __getattr__(self, name):
        from exp3_b200 import paged
        return getattr(paged, name)

    @staticmethod
    def paged_append(k, v, pool, page_table, starts, counts=None, q=None, rope=None, q_out=None, k_out=None):
        d, half = k.shape[-1], k.shape[-1] // 2

        def turn(x, positions):
            c, s = rope[positions, None, :half], rope[positions, None, half:]
            a, b = x[..., :half].float(), x[..., half:].float()
            return torch.cat((a * c - b * s, b * c + a * s), -1).to(x.dtype)

        for b in range(k.shape[0]):
            if starts[b] < 0:
                continue
            at = int(starts[b]) + torch.arange(k.shape[1])
            page, row = _rows(page_table, pool, b, at)
            kr = turn(k[b], at)
            pool[page, :, row, :d], pool[page, :, row, d:] = kr, v[b]
            if k_out is not None:
                k_out[b] = kr
            if q is not None:
                q_out[b] = turn(q[b], at)
        return q_out

    @staticmethod
    def paged_gather(pool, page_table, starts, counts, length, k_out=None, v_out=None):
        d = pool.shape[-1] // 2
        for b in range(starts.shape[0]):
            page, row = _rows(page_table, pool, b, int(starts[b]) + torch.arange(length))
            k_out[b], v_out[b] = pool[page, :, row, :d], pool[page, :, row, d:]
        return k_out, v_out

    @staticmethod
    def paged_decode_attention(q, pool, page_table, starts, scale, counts=None, out=None, lse=None, ws=None):
        out = torch.zeros_like(q)
        d = q.shape[-1]
        for b in range(q.shape[0]):
            if starts[b] < 0:
                continue
            n = int(starts[b]) + q.shape[1]
            page, row = _rows(page_table, pool, b, torch.arange(n))
            out[b] = causal(q[b], pool[page, :, row, :d], pool[page, :, row, d:], scale)
        return out


def causal(q, k, v, scale):
    """q [L, H, d]: the last L rows of k, v [n, Hkv, d]."""
    group, n = q.shape[1] // k.shape[1], k.shape[0]
    s = torch.einsum("lhd,nhd->hln", q.double(), k.double().repeat_interleave(group, 1)) * scale
    first = n - q.shape[0]
    s = s.masked_fill(torch.arange(n) > first + torch.arange(q.shape[0])[:, None], float("-inf"))
    return torch.einsum("hln,nhd->lhd", s.softmax(-1), v.double().repeat_interleave(group, 1)).to(q.dtype)


class PlainOps:
    BLOCK_SIZE = 128

    @staticmethod
    def prefill_attention(q, k, v, method, alpha, scale, sink, window, last_full, out=None, tile_range=None):
        assert method == "dense"
        first = 128 * tile_range[0] if tile_range else 0
        out = torch.full_like(q, float("nan"))
        out[0, first:] = causal(q[0, first:], k[0], v[0], scale)
        return out


class PlainModel(Qwen2Model):
    def __init__(self, **kw):
        super().__init__(CFG, device="cpu", attention=AttentionSettings("dense"), **kw)
        self.peer_all_reduce = False

    def _rmsnorm(self, x, weight, residual=None):
        if residual is not None:
            residual += x
            x = residual
        x = x.float()
        return (x * (x.square().mean(-1, keepdim=True) + self.cfg.rms_norm_eps).rsqrt()).to(weight.dtype) * weight

    def _silu_mul(self, gu):
        gate, up = gu.float().chunk(2, -1)
        return (torch.nn.functional.silu(gate) * up).to(gu.dtype)


def use_plain_calls(set_attribute):
    """set_attribute(module, name, value): pytest's monkeypatch.setattr, or setattr in a process of its own."""
    set_attribute(model_module, "paged", PlainPaged())
    set_attribute(model_module, "ops", PlainOps)


def prompt(n, seed):
    return torch.randint(0, CFG.vocab_size, (n,), generator=torch.Generator().manual_seed(seed))
