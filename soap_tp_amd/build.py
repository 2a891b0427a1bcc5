"""Compile the gfx950 kernels into ``soap_tp_amd/libsoap_mi355.so`` with hipcc.

Run as ``python -m soap_tp_amd.build``.  hipcc cross-compiles without a GPU, so this works
on a build host; the resulting shared library is loaded with ctypes by ``soap_tp_amd._native``.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess
import sys
import tempfile
from concurrent.futures import ThreadPoolExecutor
from pathlib import Path
from typing import List

PACKAGE_DIR = Path(__file__).resolve().parent
CSRC_DIR = PACKAGE_DIR / "csrc"
LIBRARY_PATH = PACKAGE_DIR / "libsoap_mi355.so"
INCLUDE_DIR = PACKAGE_DIR.parent / "include"
# A C++ program that calls the C ABI without Python or torch (used by a GPU test and for
# hardware-counter runs, where the profiled program should be a plain executable).
ABI_PROBE_SOURCE = PACKAGE_DIR.parent / "tests" / "native" / "abi_probe.cpp"
ABI_PROBE_PATH = PACKAGE_DIR.parent / "tests" / "native" / "abi_probe.bin"
SOURCES = ("api.hip", "products.hip", "products_f32.hip", "products_bf16.hip", "products_f16.hip", "products_i8.hip")

# -packed-fp32-ops is switched off on purpose: the compiler must not fuse scalar fp32 code
# into v_pk_* instructions on this target.
HIPCC_FLAGS = (
    "--offload-arch=gfx950",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-Wno-unused-result",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
)


def hipcc_path() -> str:
    found = shutil.which("hipcc") or "/opt/rocm/bin/hipcc"
    if not os.path.exists(found):
        raise RuntimeError("hipcc was not found; the gfx950 kernels cannot be built.")
    return found


def _run(command, verbose: bool) -> None:
    if verbose:
        print(" ".join(command), flush=True)
    completed = subprocess.run(command, capture_output=True, text=True)
    noise = "'-packed-fp32-ops' is not a recognized feature"
    stderr = "\n".join(line for line in completed.stderr.splitlines() if noise not in line)
    if completed.returncode != 0:
        raise RuntimeError(f"hipcc failed ({completed.returncode}):\n{stderr}")
    if verbose and stderr.strip():
        print(stderr, file=sys.stderr)


def _scalar_registers(operands: str) -> set:
    found = set()
    for first, last, single in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b", operands):
        found.update(range(int(first), int(last) + 1) if first else [int(single)])
    return found


def unsettled_loads(listing: str) -> List[str]:
    """Loads to LDS in a disassembly that read a scalar register less than five wait states after a vector
    instruction wrote it.  The products' kernels have these loads in inline assembly (load_to_lds in
    csrc/products.hpp), where the compiler does not see to that, and the hardware does not either."""
    code, at_address, jumps = [], {}, {}  # (name, operands, first in its function), by address; jumps to an address
    first = True
    for line in listing.splitlines():
        match = re.match(r"\s+(\w+)\s*(.*?)\s*// ([0-9A-F]+):", line)
        if not match:
            first = True
            continue
        name, operands, address = match.group(1), match.group(2), int(match.group(3), 16)
        if name == "s_branch" or name.startswith("s_cbranch"):
            jump = int(operands.split()[0])
            jumps.setdefault(address + 4 + 4 * (jump - 65536 if jump >= 32768 else jump), []).append(len(code))
        at_address[address] = len(code)
        code.append((name, operands, first))
        first = False
    before = {at_address[address]: sources for address, sources in jumps.items() if address in at_address}

    def written_near(at: int, states: int, read: set) -> bool:
        """Whether a vector instruction wrote one of the registers within so many wait states before ``at``."""
        falls_in = [] if code[at][2] or code[at - 1][0] in ("s_branch", "s_endpgm", "s_setpc_b64") else [at - 1]
        for source in falls_in + before.get(at, []):
            name, operands, _ = code[source]
            results = 2 if re.search("_co_|div_scale|mad_[iu]64", name) else 1  # (the second is a carry or a flag)
            if name.startswith("v_") and _scalar_registers(",".join(operands.split(",")[:results])) & read:
                return True
            left = states - 1 - (int(operands) if name == "s_nop" else 0)
            if left > 0 and written_near(source, left, read):
                return True
        return False

    return [f"{name} {operands}" for at, (name, operands, _) in enumerate(code)
            if name.startswith("buffer_load") and operands.endswith(" lds") and written_near(at, 5, _scalar_registers(operands))]


def check_loads(library: Path) -> int:
    """Raise if a kernel of the library has an unsettled load, or has loads to LDS and spills registers (a
    spilled scalar register comes back through a vector instruction).  Returns how many such loads there are."""
    places = (Path(os.path.realpath(hipcc_path())).parent.parent / "llvm" / "bin", Path("/opt/rocm/llvm/bin"))
    tools = next((place for place in places if (place / "llvm-objdump").exists()), None)
    if tools is None:
        raise RuntimeError("llvm-objdump was not found; the loads to LDS cannot be checked.")
    loads = 0
    with tempfile.TemporaryDirectory(prefix="soap_mi355_") as folder:
        (Path(folder) / "library.so").symlink_to(Path(library).resolve())

        def output(tool: str, *arguments: str) -> str:
            return subprocess.run([str(tools / tool), *arguments], cwd=folder, check=True, capture_output=True, text=True).stdout

        output("llvm-objdump", "--offloading", "library.so")
        for part in sorted(Path(folder).glob("library.so.*gfx950")):
            listing = output("llvm-objdump", "-d", part.name)
            here = len(re.findall(r"^\s+buffer_load\w* .* lds\b", listing, flags=re.M))
            if here == 0:
                continue
            loads += here
            unsettled = unsettled_loads(listing)
            if unsettled:
                raise RuntimeError(f"{len(unsettled)} loads to LDS read a scalar register too soon, the first: {unsettled[0]}")
            spills = re.findall(r"\.[sv]gpr_spill_count: *(\d+)", output("llvm-readelf", "--notes", part.name))
            if not spills or set(spills) != {"0"}:
                raise RuntimeError("kernels with loads to LDS spill registers")
    return loads


def build(verbose: bool = False) -> Path:
    """Compile the sources side by side, link them and check the loads to LDS."""
    hipcc = hipcc_path()
    with tempfile.TemporaryDirectory(prefix="soap_mi355_") as folder:
        objects = [str(Path(folder) / f"{Path(source).stem}.o") for source in SOURCES]
        commands = [[hipcc, *HIPCC_FLAGS, "-c", str(CSRC_DIR / source), "-o", target]
                    for source, target in zip(SOURCES, objects)]
        with ThreadPoolExecutor(max_workers=min(len(commands), os.cpu_count() or 1)) as pool:
            list(pool.map(lambda command: _run(command, verbose), commands))
        linked = LIBRARY_PATH.with_name(f"{LIBRARY_PATH.stem}.new.so")
        try:
            _run([hipcc, "--offload-arch=gfx950", "-shared", *objects, "-o", str(linked)], verbose)
            check_loads(linked)
            os.replace(linked, LIBRARY_PATH)
        finally:
            linked.unlink(missing_ok=True)
    return LIBRARY_PATH


def build_abi_probe(verbose: bool = False) -> Path:
    """Host-only build of tests/native/abi_probe.cpp against the shared library."""
    command = [hipcc_path(), "-O2", "-std=c++17", "-I", str(INCLUDE_DIR), str(ABI_PROBE_SOURCE),
               "-L", str(PACKAGE_DIR), "-lsoap_mi355", "-Wl,-rpath,$ORIGIN/../../soap_tp_amd",
               "-Wno-unused-result", "-o", str(ABI_PROBE_PATH)]
    if verbose:
        print(" ".join(command), flush=True)
    completed = subprocess.run(command, capture_output=True, text=True)
    if completed.returncode != 0:
        raise RuntimeError(f"hipcc failed ({completed.returncode}):\n{completed.stderr}")
    return ABI_PROBE_PATH


if __name__ == "__main__":
    print(build(verbose=True))
    print(build_abi_probe(verbose=True))
