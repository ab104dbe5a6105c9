"""What masked attention's planner decides (tests/cpp/masked_plan_query.cpp, built by
__graft_entry__.build(); no GPU), and calls that reach everything it can decide."""
import os
import subprocess

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "masked_plan_query")
CUS = 256  # compute units of an MI355X


def built():
    return os.path.exists(BIN)


def ask(shapes):
    """An answer to each (batch, heads, kv_heads, seq_q, seq_k, d_head), as text."""
    out = subprocess.run([BIN], input="".join(" ".join(map(str, s)) + f" {CUS}\n" for s in shapes),
                         capture_output=True, text=True, timeout=60, check=True)
    return out.stdout.splitlines()


def kernels(shape, answer):
    """The kernels of a call, forward and backward: which, of what width, over heads that
    fill it or not, and whether workgroups share its work."""
    d = shape[5]
    forward, shared, q_parts, kv_parts, _, _ = answer.split()
    column = next(n for n in (1, 2, 4, 8) if d <= 16 * n)  # times 16 columns
    width = next(n for n in (32, 64, 96, 128) if d <= n)
    fill = "whole" if d == width else "part"
    spread = lambda n: "shared" if int(n) > 1 else "alone"
    if forward == "rows":
        yield f"rows {column} {spread(shared)}"
    else:
        yield f"{forward} {width} {fill} {spread(shared)}"
    yield f"backward {width} {fill} dq {spread(q_parts)}"
    yield f"backward {width} {fill} dk dv {spread(kv_parts)}"


EVERY = ({f"rows {c} {s}" for c in (1, 2, 4, 8) for s in ("alone", "shared")}
         | {f"tiles128 {w} {f} {s}" for w in (32, 64, 96, 128) for f in ("whole", "part")
            for s in ("alone", "shared")}
         | {f"tiles256 {w} {f} {s}" for w in (32, 64, 96, 128) for f in ("whole", "part")
            for s in ("alone", "shared")}
         | {f"backward {w} {f} {g} {s}" for w in (32, 64, 96, 128) for f in ("whole", "part")
            for g in ("dq", "dk dv") for s in ("alone", "shared")})

SHAPES = []
for _d in (32, 24, 64, 40, 96, 70, 128, 100):
    SHAPES += [
        (2, 3, 3, 150, 150, _d),       # short walks
        (1, 1, 1, 2500, 2500, _d),     # few units: walks in parts
        (1, 2, 1, 40, 5000, _d),       # a long side of keys,
        (1, 4, 1, 1500, 30, _d),       # of rows
        (8, 16, 16, 1500, 1500, _d),   # many units
        (1, 4, 4, 12000, 12000, _d),   # and fewer of 256 rows than workgroups at once
        (32, 32, 32, 700, 1000, _d),   # and more
    ]
for _d in (16, 5, 32, 64, 128, 77):
    SHAPES += [(3, 4, 2, 1, 200, _d), (3, 4, 2, 1, 3000, _d), (2, 8, 1, 3, 700, _d)]
