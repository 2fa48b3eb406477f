"""From an encoder's hidden states to search results, with an 8-bit head and an 8-bit store of the embeddings.

    python examples/q8_embedding_search.py [--n 20000] [--nq 256]

The head is the encoder's last norm (with its residual) and a projection whose weights are held in 8 bits. Its
embeddings are indexed; they are also kept as 8-bit rows, from which the index's candidates are read back and ordered
by exact inner product. Hidden states are synthetic: each query is a base item's, with noise."""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import jhq_gpu_b200 as J


def empty_q8(rows, dim):
    """int8 rows that begin on 16-byte boundaries, and their scales."""
    q = torch.empty(rows, -(-dim // 16) * 16, dtype=torch.int8, device="cuda")[:, :dim]
    return q, torch.empty(rows, device="cuda")


class Head:
    """RMS norm and 8-bit projection: hidden states (and a residual) to float32 embeddings."""

    def __init__(self, norm_weight, projection):
        self.norm_weight = norm_weight
        self.w, self.w_scale = empty_q8(*projection.shape)
        J.q8_write(J.View.of(projection), J.Q8Rows.of(self.w, self.w_scale), stream=stream())

    def __call__(self, x, residual):
        """Embeddings; `residual` becomes x + residual."""
        q, scale = empty_q8(*x.shape)
        out = torch.empty(len(x), len(self.w), device="cuda")
        rows, r = J.Q8Rows.of(q, scale), J.View.of(residual)
        J.q8_rms_norm(J.View.of(x), rows, weight=J.View.of(self.norm_weight), residual=r, residual_out=r, stream=stream())
        J.q8_matmul(rows, J.Q8Rows.of(self.w, self.w_scale), J.View.of(out), stream=stream())
        return out


def stream():
    return torch.cuda.current_stream().cuda_stream


def main(n=20000, nq=256, hidden=512, dim=128, k=10, seed=0):
    """Share of the queries whose first result is the item that they were made from."""
    g = torch.Generator("cuda").manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    head = Head((1 + 0.1 * randn(hidden)).bfloat16(), randn(dim, hidden).bfloat16())
    x, residual = randn(n, hidden).bfloat16(), randn(n, hidden).bfloat16()
    source = torch.randint(0, n, (nq,), generator=g, device="cuda")
    qx, q_residual = (x[source] + 0.1 * randn(nq, hidden)).bfloat16(), residual[source].clone()

    base = head(x, residual)
    base /= base.norm(dim=1, keepdim=True)
    index = J.JHQGpuIndex(dim, J.Params(M=dim // 4, nlist=1, nprobe=1, batch_size=nq))
    host = base.cpu().numpy()
    index.train(host)
    index.add(host)
    kept, kept_scale = empty_q8(n, dim)
    J.q8_write(J.View.of(base), J.Q8Rows.of(kept, kept_scale), stream=stream())

    query = head(qx, q_residual)
    query /= query.norm(dim=1, keepdim=True)
    dists, ids = torch.empty(nq, k, device="cuda"), torch.empty(nq, k, dtype=torch.int32, device="cuda")
    index.search_device(query.data_ptr(), nq, k, dists.data_ptr(), ids.data_ptr(), stream())
    found = torch.empty(nq * k, dim, device="cuda")           # a missing result's id is -1 and reads as zeros
    slots = ids.long().view(-1)                               # lives until the read has run
    J.q8_read(J.Q8Rows.of(kept, kept_scale), J.View.of(found), slots=slots, stream=stream())
    score = (found.view(nq, k, dim) * query[:, None]).sum(2)
    first = ids.long().gather(1, score.argmax(1, keepdim=True))[:, 0]
    torch.cuda.current_stream().synchronize()
    index.check_device_status()
    J.q8_check_status()
    return float((first == source).float().mean())


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--n", type=int, default=20000)
    ap.add_argument("--nq", type=int, default=256)
    a = ap.parse_args()
    print(f"first result is the query's own item: {main(a.n, a.nq):.4f} of {a.nq} queries over {a.n} items")
