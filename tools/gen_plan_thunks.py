"""Generates cap2det_amd/csrc/plan_thunks.inc from the headers under include/: one typed thunk per C-ABI
entry point, `int thunk(const long long* v)`, that unpacks the recorded argument words into the
entry point's own parameter types (pointers and integers from the 64-bit word, floats from its low
32 bits) — the step plan of csrc/plan.hip calls entry points through these, never through a guessed
calling convention.  Run by the Makefile; the output is not committed.

  python tools/gen_plan_thunks.py include/cap2det_hip.h include/cap2det_products.h cap2det_amd/csrc/plan_thunks.inc
"""
import re
import sys


def main():
  headers, out = sys.argv[1:-1], sys.argv[-1]
  text = re.sub(r"/\*.*?\*/", "", "\n".join(open(h).read() for h in headers), flags=re.S)
  lines = ["// GENERATED by tools/gen_plan_thunks.py from the headers under include/ — do not edit.", ""]
  table = []
  for m in re.finditer(r"(const char\*|unsigned long long|unsigned int|long long|int)\s+(c2dp?_\w+)"
                       r"\s*\(([^)]*)\)\s*;", text):
    ret, name, params = m.group(1), m.group(2), m.group(3).strip()
    if ret != "int" or name.startswith("c2d_plan_"):
      continue                      # (queries that return a value, and the plan's own interface)
    args = []
    plist = [] if params in ("void", "") else [p.strip() for p in params.split(",")]
    for i, p in enumerate(plist):
      t = re.sub(r"\b[A-Za-z_]\w*$", "", p).strip() if (" " in p or "*" in p) else p
      if "*" in t:
        args.append("(%s)(uintptr_t)v[%d]" % (t, i))
      elif t == "float":
        args.append("plan_f32(v[%d])" % i)
      elif t in ("int", "long long", "unsigned long long", "unsigned int", "int32_t"):
        args.append("(%s)v[%d]" % (t, i))
      else:
        raise SystemExit("gen_plan_thunks: parameter type %r of %s" % (t, name))
    lines.append("static int thunk_%s(const long long* v) { (void)v; return %s(%s); }"
                 % (name, name, ", ".join(args)))
    table.append('  {"%s", thunk_%s, %d},' % (name, name, len(plist)))
  lines += ["", "static const PlanThunk kPlanThunks[] = {"] + table + ["};", ""]
  with open(out, "w") as f:
    f.write("\n".join(lines))


if __name__ == "__main__":
  main()
