"""Encoder forward on the GPU and end-to-end queries/s including the encode.

For each architecture (all-MiniLM-L6-v2: 6 x 384; all-mpnet-base-v2 sized: 12 x 768), seeded
random weights (no checkpoint offline — the forward is the real one, the vectors are not):
  * corpus encode: N node texts shaped like build_vector_index's ("Entity: {name}. {desc}",
    hierarchical_graph.py:574) -> texts/s, tokens/s, and the transformer's matmul TFLOP/s;
  * query path at C2 (d = 768 only): B = 1024 query texts -> GPU encode -> fused top-10 over the
    90k x 768 bf16 index, one step = encode + search, queries/s (the BASELINE metric's path with
    the encoder included; bench.py's headline excludes it).
Prints one JSON line.
"""
import argparse
import json
import os
import sys
import time

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [os.path.join(ROOT, "ah-rag_amd"), ROOT]

import numpy as np  # noqa: E402
import torch  # noqa: E402

from ah_rag.embeddings import DenseIndex  # noqa: E402
from ah_rag.encoder import ARCHS, TorchEncoder  # noqa: E402
from ah_rag.synthetic import HOTPOT_90K, SyntheticCorpus  # noqa: E402

WORDS = ("film director river city album band war novel bridge station king queen born american "
         "british singer actor football club season team village county district university "
         "school church museum park lake mountain island railway company founded known").split()


def texts(n, seed, lo=8, hi=48):
    rng = np.random.default_rng(seed)
    out = []
    for _ in range(n):
        name = " ".join(w.capitalize() for w in rng.choice(WORDS, size=2))
        desc = " ".join(rng.choice(WORDS, size=int(rng.integers(lo, hi))))
        out.append(f"Entity: {name}. {desc}.")
    return out


def flops_per_token(a, seq):
    h, L, f = a["hidden_size"], a["num_hidden_layers"], a["intermediate_size"]
    return 2 * L * (4 * h * h + 2 * h * f) + 2 * L * 2 * seq * h  # projections + FFN + QK^T, PV


def timed(fn, reps):
    fn()
    torch.cuda.synchronize()
    t0 = time.perf_counter()
    for _ in range(reps):
        fn()
    torch.cuda.synchronize()
    return (time.perf_counter() - t0) / reps


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--corpus", type=int, default=20000)
    ap.add_argument("--batch", type=int, default=1024)
    ap.add_argument("--reps", type=int, default=3)
    ap.add_argument("--packed", action="store_true", help="batches without padding (ah_rag.packed_encoder)")
    a = ap.parse_args()
    dev = torch.device("cuda", 0)
    out = {"weights": "seeded random (no checkpoint offline); forward, shapes and sequence lengths are the real ones"}
    corpus_texts = texts(a.corpus, 1)
    for model in ("all-MiniLM-L6-v2", "all-mpnet-base-v2"):
        enc = TorchEncoder(model, dev, packed=a.packed)
        ntok = sum(len(t) for t in enc.tokenizer(corpus_texts))
        seq = ntok / len(corpus_texts)
        dt = timed(lambda: enc.encode(corpus_texts, normalize_embeddings=True, convert_to_tensor=True), a.reps)
        tf = flops_per_token(ARCHS[model], seq) * ntok / dt / 1e12
        out[model] = {"dim": enc.dim, "corpus_texts": len(corpus_texts), "mean_tokens": round(seq, 1),
                      "texts_per_s": round(len(corpus_texts) / dt, 1), "tokens_per_s": round(ntok / dt, 1),
                      "transformer_tflops": round(tf, 1), "batch_size": 256}
        if enc.dim == 768:
            c = SyntheticCorpus(HOTPOT_90K, dev)
            rows = c.rows()
            ix = DenseIndex(768, rows.shape[0], dtype="bf16", device=dev)
            ix.upsert(rows)
            ix.reserve(a.batch, 10)
            qt = texts(a.batch, 2, 2, 12)  # short query texts

            def step():
                q = enc.encode(qt, normalize_embeddings=True, convert_to_tensor=True, batch_size=a.batch)
                return ix.query(q, 10)

            dt_e2e = timed(step, max(5, a.reps))
            qv = enc.encode(qt, normalize_embeddings=True, convert_to_tensor=True, batch_size=a.batch)
            dt_search = timed(lambda: ix.query(qv, 10), 20)
            out["c2_end_to_end"] = {"model": model, "batch": a.batch, "queries_per_s": round(a.batch / dt_e2e, 1),
                                    "ms_per_step": round(dt_e2e * 1e3, 3),
                                    "search_only_ms": round(dt_search * 1e3, 3),
                                    "encode_ms": round((dt_e2e - dt_search) * 1e3, 3)}
            ix.close()
        del enc
        torch.cuda.empty_cache()
    print(json.dumps(out), flush=True)


if __name__ == "__main__":
    main()
