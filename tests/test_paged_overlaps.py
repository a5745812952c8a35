"""Calls over a paged cache whose outputs overlap what they read are refused, on the
host and before any launch, and columns of one buffer that do not overlap are not.
No GPU needed (the pointers below are never followed)."""
import odiengine_b200 as ob

from test_paged_refusals import NEED, append, attend, batch, cache, refused, step, tables


def overlapping(**kw):
    """Sizes and addresses that do not overlap, but for what is asked."""
    at = {k: 0x10000000 * (i + 1) for i, k in enumerate(
        ("k", "v", "table", "tlens", "free", "count", "starts", "blens", "positions", "slots", "work", "q", "out", "slopes", "scratch"))}
    return at | kw


def test_an_attention_output_over_what_the_call_reads_is_refused():
    one = 2 * 10 * 2 * 16 * 128  # bytes of k, and of v
    for what, end in (("k", one), ("v", one), ("scratch", NEED), ("slopes", 4 * 6), ("q", 2 * 768 * 4)):
        for off in (0, end - 4, 4 - 4 * 768 * 2):  # its first row, its last value, the output's last
            a = overlapping()
            c, t = cache(k=a["k"], v=a["v"]), tables(a["table"], a["tlens"], a["free"], a["count"])
            b = batch(a["starts"], a["blens"], a["positions"], a["slots"], a["work"])
            refused(attend(c, t, b, q=a["q"], out=a[what] + off, slopes=a["slopes"], scr=a["scratch"]), word="overlaps")


def test_an_append_over_the_cache_is_refused():
    one = 2 * 10 * 2 * 16 * 128
    a = overlapping()
    b = batch(a["starts"], a["blens"], a["positions"], a["slots"], a["work"])
    for what in ("k", "v"):
        for off in (0, one - 4, 4 - 4 * 768 * 2):
            refused(append(cache(k=a["k"], v=a["v"]), b, qkv=a["q"], out=a[what] + off), word="overlaps")
            refused(append(cache(k=a["k"], v=a["v"]), b, qkv=a[what] + off, out=a["out"]), word="overlaps")


def test_verify_outputs_over_what_the_call_reads_are_refused():
    n = ob.lib().odi_cuda_verify_scratch_bytes(5, 2, 100)
    at = {k: 0x10000000 * (i + 1) for i, k in enumerate(("x", "tok", "st", "p", "ua", "un", "acc", "nxt", "scr"))}

    def call(**kw):
        a = at | kw
        return ob.lib().odi_cuda_verify_sampled(a["x"], 100, a["tok"], a["st"], 5, 2, 100, 1.0, a["p"], 100, a["ua"], a["un"], a["acc"],
                                                a["nxt"], a["scr"], n, None)

    for out in ("acc", "nxt"):
        for what, end in (("x", 2000), ("tok", 20), ("st", 12), ("p", 2000), ("ua", 20), ("un", 8), ("scr", n), ("nxt" if out == "acc" else "acc", 8)):
            for off in (0, end - 4, -4):
                refused(call(**{out: at[what] + off}), word="overlap")


def test_step_lists_over_what_a_step_writes_are_refused():
    a = overlapping(new=0x7F0000000)
    t = tables(a["table"], a["tlens"], a["free"], a["count"])
    b = batch(a["starts"], a["blens"], a["positions"], a["slots"], a["work"])
    for k in ("keep", "new", "prefix"):
        for what, end in (("table", 4 * 3 * 4), ("free", 4 * 10)):
            for off in (0, end - 4, -8):
                refused(step(t, b, **({"new": a["new"]} | {k: a[what] + off})), word="overlaps")
    for what, end in (("tlens", 12), ("count", 4), ("starts", 16), ("blens", 12), ("positions", 160), ("slots", 160)):
        for off in (0, end - 4, -8):
            refused(step(t, b, new=a["new"], prefix=a[what] + off), word="overlaps")
