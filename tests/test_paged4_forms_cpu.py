"""Which form of the kernel of few rows over pages of 4 bits each call of paged4_variants
takes: the launch's own rule, asked on the host."""
from paged4_variants import (CALLS, EIGHT, EIGHT_SPLIT, FOUR, MISSING, MISSING_WINDOWS, PAGE, STALE, UNSEEN,
                             UNSEEN_WINDOWS, WIDE, WIDE_SPLIT, Call)
from test_paged_share_cpu import _run


def test_forms(tmp_path):
    body = []
    others = [Call(form, heads, 2, 96, (length + more,), (n,), *window)
              for calls, windows, more in ((UNSEEN, UNSEEN_WINDOWS, STALE), (MISSING, MISSING_WINDOWS, 0))
              for heads, n, length, form in calls for window in windows]
    for c in CALLS + others:
        tile, wide, is_split = c.form
        body.append(f"  {{ const Plan p = plan(4, {len(c.new)}, {sum(c.new)}, {c.heads}, {c.kv_heads}, {PAGE}, "
                    f"{c.width}, {c.window or 'INT32_MAX'}, {c.sinks});\n"
                    f"    if (p.tile != {tile} || p.wide != {int(wide)} || (p.splits > 1) != {int(is_split)}) {{\n"
                    f'      std::printf("{c}: tile %d, wide %d, splits %d\\n", p.tile, p.wide, p.splits);\n'
                    f"      ++split;\n    }} }}")
    _run(tmp_path, "\n".join(body) + "\n  return split > 0;")
    for form in (FOUR, WIDE, WIDE_SPLIT, EIGHT, EIGHT_SPLIT):
        for d in (64, 96, 128):
            assert sum(c.form == form and c.d == d for c in CALLS) >= 6
