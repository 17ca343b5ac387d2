"""Small calls that reach every launch of the paged attention and of the log
probabilities: test_paged_plans.py holds the rules to the launches named here,
test_gpu_paged_launches.py runs them."""

FORMATS = ["f32", "f16", "q8_0", "q4_0"]


def ragged(n, most, longest):
    """Lengths up to `most`: empty sequences first, last and in runs, and one long one."""
    lengths = [0 if i < 3 or i >= n - 2 or i // 9 % 4 == 1 else 1 + 53 * i % most for i in range(n)]
    lengths[n // 2] = longest
    return lengths


def attention():
    """name: (format, q heads, KV heads, head_dim, page size, table width, lengths, window, launch)."""
    cases = {}
    for fmt in FORMATS:
        # split rows of more sequences than a wavefront, than a chunk of them and than two, joined by 256 threads
        for n in (65, 256, 257, 600):
            for H, KH, D in ((8, 2, 64), (8, 1, 128), (16, 1, 256)):
                cases[f"split_{fmt}_{n}_{D}"] = (fmt, H, KH, D, 16, 2048, ragged(n, 110, 1500), 0,
                                                 ("split", "wave" if n <= 64 else "chunk" if n <= 256 else "chunks",
                                                  (16 if D == 64 else 32 if D == 128 else 64, 256)))
        # parts of several units, of which some have one more
        cases[f"parts_{fmt}"] = (fmt, 6, 2, 96, 64, 512, [(97 * i) % 701 for i in range(300)], 0, ("split", "chunks", (32, 256)))
        # of sequences whose heads are two rows; windows that begin inside units
        cases[f"tiles_{fmt}"] = (fmt, 20, 1, 160, 16, 2048, ragged(270, 90, 777), 0, ("split", "chunks", (64, 256)))
        cases[f"window_{fmt}"] = (fmt, 8, 1, 256, 16, 8192, ragged(90, 300, 9000), 6000, ("split", "chunk", (64, 256)))
        # few query rows
        cases[f"few_{fmt}"] = (fmt, 4, 2, 64, 16, 2048, ragged(70, 200, 1200), 0, ("split", "chunk", (16, 1024)))
        cases[f"fewer_{fmt}"] = (fmt, 8, 1, 160, 64, 800, [700, 0, 33], 0, ("split", "wave", (8, 1024)))
        # whole rows: short ones, some of them, more than there are CUs
        cases[f"short_{fmt}"] = (fmt, 8, 2, 64, 16, 6, ragged(20, 96, 96), 0, ("whole", 4))
        cases[f"some_{fmt}"] = (fmt, 8, 2, 64, 16, 24, ragged(20, 384, 384), 0, ("whole", 16))
        cases[f"some_wide_{fmt}"] = (fmt, 8, 1, 192, 16, 24, ragged(70, 384, 384), 0, ("whole", 6 if fmt == "f16" else 8))
        cases[f"many_{fmt}"] = (fmt, 8, 2, 128, 16, 24, ragged(140, 384, 384), 0, ("whole", 4))
    return cases


ATTENTION = attention()

# name: (rows, vocabulary, padding of a row, strips of a slice, whether a wavefront has more than one slice, threads of a row)
LOGPROBS = {
    "one_strip": (5, 900, 0, 1, False, 1024),
    "one_strip_each": (255, 32001, 3, 1, False, 1024),
    "two_strips": (40, 262144, 0, 2, False, 1024),
    "two_strips_again": (80, 262144, 1, 2, True, 1024),
    "two_strips_odd": (512, 16385, 0, 2, False, 1024),
    "more_rows": (600, 16385, 2, 2, False, 256),
    "more_rows_again": (1100, 16385, 0, 2, True, 256),
    "rows_of_one_slice": (9000, 1025, 0, 2, True, 256),
    "rows_of_less_than_a_strip": (9001, 130, 5, 2, True, 256),
    "rows_of_a_strip_each": (700, 5000, 0, 1, False, 256),
}
