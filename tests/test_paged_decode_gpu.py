"""GPU: the decode forward pass (nedo_gpu_decoder_*) against the same pass with its cache and
attention replaced by the paged operators: one sequence, F32 pages dealt out in no order, the
model's sliding window.  Every pass's logits agree within what test_decoder_gpu.py allows against the
reference.  (The append forms its angles in 64 bits, the decode pass in 32 as the reference does: at
these positions, below 100, that is a turn of at most 100 * 2^-24 radians.)"""
import os
import sys

import numpy as np
import pytest

from conftest import ROOT

sys.path[:0] = [os.path.join(ROOT, "tests", "golden")]
import make_decode_golden as M  # noqa: E402
import nedo_gpu  # noqa: E402
from decode_oracle import DecodeOracle, _norm_weight, rms_norm  # noqa: E402
from nedo_gpu import gguf as G  # noqa: E402
from nedo_gpu.decoder import Decoder  # noqa: E402

pytestmark = pytest.mark.gpu

LOGIT_TOL = 2e-4
GOLDEN = np.load(os.path.join(ROOT, "tests", "golden", "decode_golden.npz"))
PAGE = 16


class PagedPass(DecodeOracle):
    """The decode pass with append and attention on the GPU, everything else as in the oracle."""

    def __init__(self, g, lib, torch, steps):
        super().__init__(g)
        self.lib, self.torch = lib, torch
        pages = -(-steps // PAGE)
        self.cache_of, self.keep = [], []
        for _ in range(self.layers):
            k, v = (torch.full((pages + 2, self.kv_heads, PAGE, self.hd), float("nan"), device="cuda") for _ in range(2))
            self.keep += [k, v]
            self.cache_of.append(nedo_gpu.KvCache(type=0, kv_heads=self.kv_heads, head_dim=self.hd, page_size=PAGE,
                                                  num_pages=pages + 2, k=k.data_ptr(), v=v.data_ptr(), bounds=None))
        order = np.random.default_rng(5).permutation(pages + 2)[:pages].astype(np.int32)
        self.start = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        self.len = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.table = torch.from_numpy(order).cuda()
        self.batch = nedo_gpu.KvBatch(seqs=1, tokens=1, max_q_len=1, max_kv_len=steps, max_pages=pages, shared_pages=0,
                                      q_start=self.start.data_ptr(), kv_len=self.len.data_ptr(),
                                      page_table=self.table.data_ptr())
        need = max(16, lib.paged_attention_workspace(self.cache_of[0], self.batch, self.heads, self.window))
        self.space = torch.empty(need, dtype=torch.uint8, device="cuda")
        self.q, self.out = (torch.empty((self.heads, self.hd), device="cuda") for _ in range(2))

    def attend(self, layer, qkv, pos):
        rows = self.torch.from_numpy(qkv).cuda()
        self.len[0] = pos + 1
        cache, st = self.cache_of[layer], self.torch.cuda.current_stream().cuda_stream
        self.lib.kv_append_dev(cache, self.batch, self.heads, rows.data_ptr(), self.theta, self.q.data_ptr(), st)
        self.lib.paged_attention_dev(cache, self.batch, self.heads, self.q.data_ptr(), self.out.data_ptr(), self.hd ** -0.5,
                                     self.window, self.space.data_ptr(), self.space.numel(), st)
        return self.out.cpu().numpy().reshape(-1)

    def forward(self, token, pos):
        g = self.g
        tt, shape, _, _ = g.tensors["token_embd.weight"]
        x = self.o.embedding_row(tt, shape[1], shape[0], g.view("token_embd.weight"), token)
        for li in range(self.layers):
            p = f"blk.{li}."
            xn = rms_norm(x, _norm_weight(g, p + "attn_norm.weight"), self.eps)
            qkv = np.concatenate([self._mv(p + f"attn_{n}.weight", xn) for n in "qkv"])
            x = (x + self._mv(p + "attn_output.weight", self.attend(li, qkv, pos))).astype(np.float32)
            xn = rms_norm(x, _norm_weight(g, p + "ffn_norm.weight"), self.eps)
            gate, up = self._mv(p + "ffn_gate.weight", xn), self._mv(p + "ffn_up.weight", xn)
            gate = ((gate / (np.float32(1.0) + np.exp(-gate))) * up).astype(np.float32)
            layers, shared, root, suffix = self.morph
            if self.route is not None and li >= self.layers - layers:
                if self.route[2 * token] < 0.5:
                    gate[shared:shared + root] = 0.0
                if self.route[2 * token + 1] < 0.5:
                    gate[shared + root:shared + root + suffix] = 0.0
            x = (x + self._mv(p + "ffn_down.weight", gate)).astype(np.float32)
        return self._mv(self.head, rms_norm(x, _norm_weight(g, "output_norm.weight"), self.eps))


@pytest.mark.parametrize("name", list(M.MODELS))
def test_paged_operators_in_the_decode_pass(lib, cuda, tmp_path, name):
    kw, prompt, _ = M.MODELS[name]
    path = str(tmp_path / (name + ".gguf"))
    G.synthetic_model(path, **kw)
    g = G.GgufFile(path)
    seq = list(prompt) + [int(i) for i in GOLDEN[name + "/ids"]]
    paged = PagedPass(g, lib, cuda, len(seq))
    dec = Decoder.from_gguf(g)
    try:
        for pos, token in enumerate(seq):
            _, want = dec.forward(token, pos)
            got = paged.forward(token, pos)
            assert np.abs(got - want).max() <= LOGIT_TOL * np.abs(want).max(), (name, pos)
        lib.status()
    finally:
        dec.close()
