"""Penalties, biases, bans and masks on logits restated in numpy: the steps of
include/backend.h in its order, each rounded to fp32, so results are exact."""
import numpy as np


def process(x, hist=None, hist_len=None, prompt_len=None, repeat=None, frequency=None, presence=None, ngram=None,
            bias_start=None, bias_id=None, bias=None, mask=None, mask_of=None):
    """(logits, ids, scores) of rows x [rows][vocab]."""
    x = x.astype(np.float32).copy()
    rows, vocab = x.shape
    one = np.float32
    ids, scores = np.full(rows, -1, np.int32), np.full(rows, -np.inf, np.float32)
    with np.errstate(all="ignore"):
        for r in range(rows):
            said = hist[r, :min(max(int(hist_len[r]), 0), hist.shape[1])] if hist is not None else np.zeros(0, np.int32)
            valid = (said >= 0) & (said < vocab)
            start = max(int(prompt_len[r]), 0) if prompt_len is not None else 0
            seen = np.unique(said[valid])
            if repeat is not None:
                v = x[r, seen]
                x[r, seen] = np.where(v > 0, v / one(repeat[r]), v * one(repeat[r]))
            t, n = np.unique(said[start:][valid[start:]], return_counts=True)
            if frequency is not None:
                x[r, t] = x[r, t] - (one(frequency[r]) * n.astype(np.float32)).astype(np.float32)
            if presence is not None:
                x[r, t] = x[r, t] - one(presence[r])
            if bias_start is not None:
                a, b = int(bias_start[r]), int(bias_start[r + 1])
                if a >= 0 and b <= len(bias_id):
                    for t, v in {int(i): v for i, v in zip(bias_id[a:b], bias[a:b])}.items():
                        if 0 <= t < vocab:
                            x[r, t] = x[r, t] + one(v)
            k = int(ngram[r]) if ngram is not None else 0
            if 1 <= k <= len(said):
                end = list(said[len(said) - k + 1:])
                for i in range(len(said) - k + 1):
                    if list(said[i:i + k - 1]) == end and 0 <= said[i + k - 1] < vocab:
                        x[r, said[i + k - 1]] = -np.inf
            if mask is not None:
                m = int(mask_of[r]) if mask_of is not None else r
                if m >= len(mask):
                    x[r] = -np.inf
                elif m >= 0:
                    ok = (mask[m][np.arange(vocab) // 32] >> (np.arange(vocab) % 32).astype(np.uint32)) & 1
                    x[r, ok == 0] = -np.inf
            fine = np.where(np.isnan(x[r]), -np.inf, x[r])
            if fine.max() > -np.inf:
                ids[r] = int(np.argmax(fine))
                scores[r] = fine.max()
    return x, ids, scores
