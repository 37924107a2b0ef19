"""Cases shared by the CPU and GPU tests of the operators for serving many sequences."""
import numpy as np

#   batch entries, beams, vocab, results
BEAM_SHAPES = [(1, 1, 1, 1), (1, 1, 7, 7), (2, 3, 5, 15), (1, 4, 32000, 8), (3, 5, 1001, 10), (7, 8, 513, 16), (2, 16, 4097, 32),
               (5, 2, 130001, 4), (1, 128, 300, 128), (4, 1, 65536, 64), (1, 8, 131072, 8)]


def beam_case(batch, beams, vocab, seed):
    """Logits with exact ties (they are fp16 anyway), masked tokens, an empty row, infinities and NaN; twin, dead and
    finished beams."""
    r = np.random.default_rng([seed, batch, beams, vocab])
    rows = batch * beams
    x = (r.standard_normal((rows, vocab)) * 3).astype(np.float16)
    x[r.random((rows, vocab)) < 0.02] = -np.inf
    s = (-12 * r.random(rows)).astype(np.float32)
    fin = np.zeros(rows, np.uint8)
    if rows >= 4:
        x[1], s[1] = x[0], s[0]                        # twins: every candidate of one ties with the other's
        s[3] = -np.inf
        fin[2] = 1
        s[2] = -1.0
    if rows >= 8:
        x[5] = -np.inf                                 # nothing left in this row
        x[6, r.integers(vocab)] = np.nan
        x[7, r.integers(vocab)] = np.inf
    return x, s, fin
