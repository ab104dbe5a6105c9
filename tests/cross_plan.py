"""What cross attention's planner decides (tests/cpp/cross_plan_query.cpp, built by
__graft_entry__.build(); no GPU), and calls that reach everything it can decide."""
import os
import subprocess

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "cross_plan_query")
CUS = 256  # compute units of an MI355X


def built():
    return os.path.exists(BIN)


def ask(shapes):
    """An answer to each (batch, heads, kv_heads, seq_q, seq_k, d_head), as text."""
    out = subprocess.run([BIN], input="".join(" ".join(map(str, s)) + f" {CUS}\n" for s in shapes),
                         capture_output=True, text=True, timeout=60, check=True)
    return out.stdout.splitlines()


def kernels(shape, answer):
    """The kernels of a call, forward and backward: which, of what width, over
    heads that fill it or not, and whether workgroups share its work."""
    _, heads, kv, seq_q, seq_k, d = shape
    forward, groups, units, backward, q_splits, kv_splits = answer.split()
    column = next(n for n in (1, 2, 4, 8) if d <= 16 * n)  # times 16 columns
    width = next(n for n in (32, 64, 96, 128) if d <= n)
    heads_fill = "whole" if d == width else "part"
    spread = lambda n: "shared" if int(n) > 1 else "alone"
    if forward == "few_keys":
        yield f"few_keys {column}"
    elif forward == "rows":
        yield f"rows {column} {spread(groups)}"
    else:
        more = "fewer" if int(units) < int(groups) else "more"
        yield f"{forward} {width} {heads_fill} " + (f"shared, {more} units" if int(groups) else "alone")
    if backward == "tiles":
        yield f"backward {width} {heads_fill} dq {spread(q_splits)}"
        yield f"backward {width} {heads_fill} dk dv {spread(kv_splits)}"
    else:
        own = seq_q * (heads // kv) if backward == "short_rows" else seq_k
        yield f"{backward} {column} x {(own + 15) // 16} {spread(max(int(q_splits), int(kv_splits)))}"


_SPREAD, _FILL = ("alone", "shared"), ("whole", "part")
EVERY = ({f"few_keys {c}" for c in (1, 2, 4, 8)}
         | {f"rows {c} {s}" for c in (1, 2, 4, 8) for s in _SPREAD}
         | {f"tiles{r} {w} {f} {s}" for r in (128, 256) for w in (32, 64, 96, 128) for f in _FILL
            for s in ("alone", "shared, fewer units", "shared, more units")}
         | {f"backward {w} {f} {g} {s}" for w in (32, 64, 96, 128) for f in _FILL
            for g in ("dq", "dk dv") for s in _SPREAD}
         | {f"short_{k} {c} x {t} {s}" for k in ("rows", "keys") for c in (1, 2, 4, 8)
            for t in (1, 2, 3) for s in _SPREAD})

# batch, heads, kv_heads, seq_q, seq_k, d_head; those of the kernels of many rows
# have several tiles of rows to an item, the last one not whole.
SHAPES = [
    (26, 4, 2, 518, 1028, 32), (6, 24, 8, 173, 1828, 32), (6, 3, 1, 1111, 3082, 32), (5, 9, 3, 1513, 907, 8),
    (10, 39, 13, 113, 601, 40), (27, 5, 5, 331, 471, 64), (1, 60, 20, 541, 1814, 8),
    (11, 13, 13, 374, 257, 128), (2, 15, 5, 2160, 299, 96), (27, 2, 2, 534, 831, 64),
    (12, 3, 3, 1799, 454, 32), (1, 6, 2, 1933, 5740, 8), (3, 60, 20, 366, 225, 96), (4, 2, 2, 797, 4065, 64),
    (2, 20, 20, 769, 865, 40), (13, 10, 5, 385, 348, 72), (2, 40, 20, 791, 243, 80), (25, 6, 2, 185, 574, 96),
    (3, 16, 8, 1386, 505, 8), (9, 13, 13, 302, 296, 128), (5, 24, 8, 537, 243, 64), (10, 9, 3, 361, 566, 72),
    (1, 8, 8, 782, 2703, 96), (5, 16, 8, 419, 397, 100), (2, 5, 5, 769, 3276, 40), (17, 8, 8, 311, 225, 100),
    (1, 40, 20, 1634, 247, 40), (2, 8, 8, 322, 2699, 72), (1, 26, 13, 258, 1710, 128),
    (3, 9, 3, 171, 2430, 100), (1, 13, 13, 2443, 229, 128), (4, 13, 13, 523, 233, 127),
    (2, 8, 8, 141, 1824, 96), (1, 2, 1, 76, 609, 32), (1, 2, 1, 73, 605, 13), (1, 1, 1, 192, 303, 128),
    (1, 1, 1, 148, 306, 127), (1, 1, 1, 148, 356, 40), (1, 1, 1, 143, 307, 72), (1, 3, 1, 47, 294, 64),
    (1, 3, 1, 11, 360, 32), (1, 3, 1, 116, 41, 8), (1, 1, 1, 281, 44, 100), (1, 2, 1, 13, 323, 64),
    (1, 1, 1, 46, 254, 100), (1, 1, 1, 275, 43, 64), (1, 2, 1, 19, 252, 64), (1, 1, 1, 250, 36, 32),
    (1, 3, 1, 85, 29, 40), (1, 2, 1, 10, 280, 8), (1, 1, 1, 24, 253, 80), (1, 3, 1, 11, 259, 8),
    (1, 1, 1, 249, 32, 24), (1, 3, 1, 7, 265, 32), (1, 1, 1, 244, 20, 96), (1, 1, 1, 165, 61, 100),
    (1, 1, 1, 252, 25, 13), (1, 1, 1, 4, 267, 8), (1, 3, 1, 2, 248, 24), (1, 3, 1, 82, 5, 32),
    (1, 2, 1, 88, 46, 40), (1, 3, 1, 82, 5, 8), (1, 1, 1, 1, 247, 64), (1, 2, 1, 121, 2, 64),
    (1, 1, 1, 242, 1, 100), (1, 1, 1, 1, 241, 128), (1, 1, 1, 192, 17, 128), (1, 1, 1, 164, 42, 16),
    (1, 2, 1, 73, 48, 32), (1, 1, 1, 143, 37, 96), (1, 1, 1, 150, 29, 72), (1, 3, 1, 51, 23, 40),
    (1, 3, 1, 47, 27, 24), (1, 2, 1, 73, 19, 8), (1, 1, 1, 54, 1, 24), (1, 1, 1, 52, 2, 13),
    (1, 1, 1, 49, 2, 96), (1, 1, 1, 49, 1, 64), (1, 1, 1, 36, 1, 32), (1, 3, 1, 12, 1, 8),
    (1, 3, 1, 11, 2, 64), (1, 1, 1, 33, 1, 80), (1, 1, 1, 19, 1, 24), (1, 1, 1, 18, 1, 64),
    (1, 3, 1, 6, 1, 8), (1, 1, 1, 17, 1, 127), (1, 1, 1, 1, 1, 72), (1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 1, 32),
    (1, 1, 1, 1, 1, 8),
]
