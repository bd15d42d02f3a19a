"""Outputs that other threads' inputs lie in are refused.  Looked at before a device is, so this needs no GPU: the addresses are never followed."""
import itertools

from test_i8_refusals import call


def meet(a, wa, lda, b, wb, ldb, rows):
    """Whether two sets of rows share an element, by looking at them all."""
    x = {a + r * lda + i for r in range(rows) for i in range(wa)}
    return any(b + r * ldb + i in x for r in range(rows) for i in range(wb))


BASE = 1 << 20  # element addresses; nothing is there


def test_rotated_queries(wf):
    """Every place of `out` beside q, k and v in units of a head's 64 elements: accepted (then the missing GPU is what ends the call) exactly where nothing is shared, where rows lie
    equally far apart; refused at the latest where they do not and their ranges meet."""
    D, far = 64, 1 << 14

    def rope(q, ldq, k, v, ldkv, out, ldo, rows, nq=2, nkv=1):
        at = [2 * (BASE + D * e) for e in (q, k, v, out)]
        rc, msg = call(wf, "wf_rope_kv_i8", at[0], ldq * D, at[1], at[2], ldkv * D, 2, 1024, 1024, 8, 0, at[3], ldo * D, 1024, 1024, 16, 16, 1, rows, nq, nkv, D, 1 << 20, 1 << 31, None)
        assert rc, "ran without a device"
        return "share" in msg

    wf_device = __import__("torch").cuda.is_available()
    if wf_device:  # a call that is accepted would be launched
        return
    for rows, out, ldo in itertools.product((1, 3), range(-12, 25), (2, 5, 6)):
        for ldq in (2, 6):
            same = out == 0 and (ldo == ldq or rows == 1)
            want = (meet(0, 2, ldq, out, 2, ldo, rows) and not same)
            got = rope(0, ldq, far, 2 * far, 1, out, ldo, rows)
            assert got >= want and (got == want or (ldo != ldq and rows > 1)), (rows, out, ldo, ldq)
        # one row: q, k, v and two columns of something else
        same = out == 0 and (ldo == 6 or rows == 1)
        want = (meet(0, 2, 6, out, 2, ldo, rows) and not same) or meet(2, 1, 6, out, 2, ldo, rows) or meet(3, 1, 6, out, 2, ldo, rows)
        got = rope(0, 6, 2, 3, 6, out, ldo, rows)
        assert got >= want and (got == want or (ldo != 6 and rows > 1)), (rows, out, ldo)


def test_attention(wf):
    import torch

    if torch.cuda.is_available():
        return
    lib, ws = wf._lib.lib(), 1 << 24

    def refused(q, out, ldq, B=2, nq=4, D=64):
        rc, msg = call(wf, "wf_attn_decode_i8", q, 2, ldq, 1024, 1024, 16, 16, None, 0, out, B, nq, 2, D, 64, 0.1, ws, lib.wf_attn_decode_i8_workspace_bytes(nq, 2, D), 0, None)
        assert rc
        return "overlap" in msg

    for ldq in (256, 300 // 8 * 8):
        end = 2 * (ldq + 256)
        for out, want in ((0, True), (end - 2, True), (end, False), (-1024 + 2, True), (-1024, False)):
            assert refused(1 << 20, (1 << 20) + out, ldq) == want, (ldq, out)
