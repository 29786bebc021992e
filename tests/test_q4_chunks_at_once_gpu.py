"""GPU: attention over 4-bit caches whose chunks the device makes as long as the lengths ask -- their length goes from
one kernel to the next through the workspace -- on several streams and in several graphs at once."""
import pytest

from q4_ref import DeviceQ4, SetupQ4

pytestmark = pytest.mark.gpu

CASES = [((12, 4, 128, 64), [5, 1, 3, 5], [20000, 5, 6400, 17777], 0), ((4, 4, 64, 64), [1] * 6, [19001, 300, 12345, 18999, 1, 17000], 0),
         ((16, 8, 128, 64), [1] * 6, [9000, 1200, 8999, 1281, 5000, 6001], 18)]


def test_several_at_once(lib, cuda):
    ds = [DeviceQ4(lib, cuda, SetupQ4(*shape, q=q, kv=kv, shared=shared, seed=51 + i)) for i, (shape, q, kv, shared) in enumerate(CASES)]
    other = [[max(1, n // 3) if n > 100 else n for n in kv] if not shared else [1152 + 20 * i for i in range(len(kv))] for _, _, kv, shared in CASES]
    need = [lib.paged_attention_workspace(d.cache, d.batch, d.s.heads) for d in ds]
    for d, n in zip(ds, need):
        assert n % (d.s.tokens * d.s.heads * (d.s.hd * 4 + 8)) == 16  # the chunks' length is there
    ws = [d.space(n) for d, n in zip(ds, need)]
    streams = [cuda.cuda.Stream() for _ in ds]
    outs = [[cuda.empty_like(d.out) for _ in range(8)] for d in ds]

    def call(i, out, stream):
        d = ds[i]
        lib.paged_attention_dev(d.cache, d.batch, d.s.heads, d.q.data_ptr(), out.data_ptr(), d.s.scale, 0, ws[i].data_ptr(), need[i],
                                stream.cuda_stream)

    call(0, outs[0][0], streams[0])  # (the library's state on the device, outside a capture)
    cuda.cuda.synchronize()
    graphs = [cuda.cuda.CUDAGraph() for _ in ds]
    for i in range(len(ds)):
        with cuda.cuda.graph(graphs[i], stream=streams[i]):
            for out in outs[i]:
                call(i, out, streams[i])
    for lens in ([c[2] for c in CASES], other):  # (other lengths: chunks of other lengths)
        for d, x in zip(ds, lens):
            d.len.copy_(cuda.tensor(x, dtype=cuda.int32))
        want = [d.attention().clone() for d in ds]
        for graphed in (False, True):
            for x in sum(outs, []):
                x.zero_()
            cuda.cuda.synchronize()
            for n in range(1 if graphed else 8):
                for i in range(len(ds)):
                    if graphed:
                        with cuda.cuda.stream(streams[i]):
                            graphs[i].replay()
                    else:
                        call(i, outs[i][n], streams[i])
            cuda.cuda.synchronize()
            for i in range(len(ds)):
                assert all(cuda.equal(out, want[i]) for out in outs[i])
    lib.status()
