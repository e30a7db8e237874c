"""Twelve passes each of the larger cases of perf/operators.py for a rocprofv3 run: `--kernel-trace --stats`, or a --pmc pass
with GRBM_GUI_ACTIVE, SQ_BUSY_CU_CYCLES, SQ_VALU_MFMA_BUSY_CYCLES, SQ_ACTIVE_INST_VALU, SQ_WAVE_CYCLES and
SQ_LDS_BANK_CONFLICT.  `run all` takes all cases.  `summarize <counter_collection.csv>` prints, per kernel and grid, the
medians of a launch: cycles, the share of them in which a CU has a wave, and of the busy CUs' SIMD cycles the shares of the matrix pipe
and of the vector unit (which run beside each other), waves a busy CU, and LDS cycles lost to bank conflicts per busy CU cycle."""
import collections, csv, os, sys

CASES = ("prompt 4x2048", "prompt long 16384", "append prefill ragged", "paged 64x8192", "paged 1x131071", "logprobs 4096x50272")


def run(which):
    import torch
    sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    from perf import operators
    operators.own = True
    for case in operators.listed():
        if which == "all" or case["name"] in CASES:
            state = operators.prepare(case, 3)
            torch.cuda.synchronize()
            for _ in range(12):
                operators.run(state)
            torch.cuda.synchronize()


def summarize(path):
    runs = collections.defaultdict(lambda: collections.defaultdict(list))
    for r in csv.DictReader(open(path)):
        if any(k in r["Kernel_Name"] for k in ("attention_p", "kv_append", "token_logprobs")):
            name = r["Kernel_Name"].replace("(anonymous namespace)::", "").replace("_ZN12_GLOBAL__N_1", "").replace("void ", "").lstrip("0123456789")
            runs[name[:44], int(r["Grid_Size"]) // int(r["Workgroup_Size"])][r["Counter_Name"]].append(float(r["Counter_Value"]))
    print(f"{'kernel':44s} {'WGs':>6s} {'launches':>8s} {'cycles':>9s} {'CU busy':>8s} {'matrix':>7s} {'vector':>7s} {'waves/CU':>8s} {'conflicts':>9s}")
    for (name, wgs), v in runs.items():
        m = {c: sorted(x)[len(x) // 2] for c, x in v.items()}
        cycles, busy = m["GRBM_GUI_ACTIVE"] / 8, m["SQ_BUSY_CU_CYCLES"]
        print(f"{name:44s} {wgs:6d} {len(v['GRBM_GUI_ACTIVE']):8d} {cycles:9.0f} {busy / (256 * cycles):8.2f} {m['SQ_VALU_MFMA_BUSY_CYCLES'] / (4 * busy):7.2f} "
              f"{m['SQ_ACTIVE_INST_VALU'] / busy:7.2f} {4 * m['SQ_WAVE_CYCLES'] / busy:8.2f} {m['SQ_LDS_BANK_CONFLICT'] / busy:9.3f}")


if __name__ == "__main__":
    summarize(sys.argv[2]) if sys.argv[1:2] == ["summarize"] else run(sys.argv[2] if sys.argv[1:2] == ["run"] and len(sys.argv) > 2 else "")
