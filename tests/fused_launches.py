"""Which kernels the products whose results are not stored as they are launch, and with what: the host side of csrc/fused*.hip and
logprobs.hip, compiled for the host alone, against a HIP runtime that runs nothing (tests/host/fused_launches.cpp)."""
import collections
import functools
import os
import re
import subprocess
import tempfile
from concurrent.futures import ThreadPoolExecutor

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "strands-decider-web_amd", "csrc")
HIPCC = "/opt/rocm/bin/hipcc"
CXX = "/opt/rocm/llvm/bin/clang++"
FILES = ("fused.hip", "fused_lanes.hip", "fused_rows.hip", "fused_tiles.hip", "fused_logits.hip", "logprobs.hip")

# kernel: its name and template arguments; rows: of the launch; the others: bytes from the call's addresses (-1: none)
Launch = collections.namedtuple("Launch", "kernel groups threads lds rows a out residual records logp lse top_ids")
Answer = collections.namedtuple("Answer", "status bytes refusal launches limits")


@functools.lru_cache(None)
def program():
    d = tempfile.mkdtemp()
    include = ["-std=c++17", "-I" + os.path.join(ROOT, "include"), "-I" + CSRC]
    exe = os.path.join(d, "launches")
    host = [CXX, "-O1", "-D__HIP_PLATFORM_AMD__", "-I/opt/rocm/include", "-Wno-unused-result", *include]
    none = os.path.join(d, "none")
    open(none, "w").close()  # (in the device code's place)
    jobs = [[HIPCC, "--offload-arch=gfx950", "--cuda-host-only", "-O1", *include, "-Xclang", "-fcuda-include-gpubinary", "-Xclang", none, "-x", "hip", "-c",
             os.path.join(CSRC, f), "-o", os.path.join(d, f + ".o")] for f in FILES]
    jobs += [host + ["-c", f, "-o", os.path.join(d, os.path.basename(f) + ".o")]
             for f in (os.path.join(CSRC, "fused_host.cpp"), os.path.join(ROOT, "tests", "host", "fused_launches.cpp"))]

    def run(cmd):
        r = subprocess.run(cmd, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr
    with ThreadPoolExecutor(4) as ex:
        list(ex.map(run, jobs))
    run([CXX, *(j[-1] for j in jobs), "-o", exe, "-lpthread"])
    return exe


def kernel(mangled):
    """fused_tiles_kernel<4, 0, 1, ...> of a mangled name."""
    m = re.match(r"_ZN2ha12_GLOBAL__N_1\d+(\w+?_kernel)I((?:L[ib]\d+E)+)E", mangled)
    return "%s<%s>" % (m.group(1), ", ".join(re.findall(r"L[ib](\d+)E", m.group(2))))


def ask(lines):
    """The answers to lines as tests/host/fused_launches.cpp takes them."""
    r = subprocess.run([program()], input="\n".join(" ".join(str(int(x) if not isinstance(x, str) else x) for x in l) for l in lines) + "\n",
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr
    answers, launches, limits, refusal = [], [], [], ""
    for line in r.stdout.splitlines():
        what, rest = line.split(" ", 1)
        if what == "refused":
            refusal = rest
        elif what == "limit":
            limits.append((kernel(rest.split()[0]), int(rest.split()[1])))
        elif what == "launch":
            n, *x = rest.split()
            launches.append(Launch(kernel(n), *map(int, x)))
        else:
            status, nbytes = map(int, rest.split())
            answers.append(Answer(status, nbytes, refusal, launches, limits))
            launches, limits, refusal = [], [], ""
    assert len(answers) == sum(l[0] != "put" for l in lines)
    return answers


def kernels():
    """All kernels of the compiled files."""
    r = subprocess.run([program()], input="kernels\n", capture_output=True, text=True, timeout=60)
    return {kernel(l.split()[1]) for l in r.stdout.splitlines()}


def put(output, base, at):
    return ("put", output, base, at)


def fused(M, N, K, fmt=(4, 32, False), gated=False, q_at=0, s_at=0):
    return ("fused", M, N, K, *fmt, gated, q_at, s_at)


def logprobs(M, V, K, fmt=(4, 32, False), n_vocab=0, targets=0, top_k=0, q_at=0, workspace=-1):
    return ("logprobs", M, V, K, *fmt, n_vocab, targets, top_k, q_at, workspace)
