"""Writes luts_data.h: the sigmoid / exp integer tables of the numerics contract
(NUMERICS.md:130, 160-161), evaluated from their definitions with Python's
round-half-even on doubles, the rounding the reference's generator uses
(python/llaccel/luts.py:18-29).  tests/test_build.py checks the header against the
committed golden tables.

Also writes device_luts.h: the same exp tables and the sampling weights' powers of two as
device data, for the calls that have no model to take its tables from."""
from __future__ import annotations

import math
from pathlib import Path


def tables():
    sig = [min(65535, round(65536.0 / (1.0 + math.exp(-(j / 16.0 - 8.0))))) for j in range(257)]
    expi = [round(65535 * math.exp(-i)) for i in range(16)]
    expf = [round(65535 * math.exp(-f / 256.0)) for f in range(256)]
    return sig, expi, expf


def render() -> str:
    sig, expi, expf = tables()
    out = ["// Generated by gen_luts.py -- integer tables of the numerics contract.", "#pragma once",
           "#include <cstdint>", "", "namespace llx {"]
    for name, vals in (("kSig", sig), ("kExpI", expi), ("kExpF", expf)):
        out.append(f"static const uint16_t {name}[{len(vals)}] = {{")
        for i in range(0, len(vals), 16):
            out.append("    " + ", ".join(str(v) for v in vals[i : i + 16]) + ",")
        out.append("};")
    out.append("}  // namespace llx")
    return "\n".join(out) + "\n"


def pow2_table():
    """2^31 * 2^(-j / 1024), j = 0..1023: no entry lies nearer than 2e-4 to a rounding tie, far
    beyond a double's error, so any platform's doubles give these integers."""
    return [round(2.0 ** 31 * 2.0 ** (-j / 1024.0)) for j in range(1024)]


def curve_table():
    """The table exponential of every index z below 4096 (NUMERICS.md:160-161)."""
    _, expi, expf = tables()
    return [(expi[z >> 8] * expf[z & 255] + 32768) >> 16 for z in range(4096)]


def render_device() -> str:
    _, expi, expf = tables()
    out = ["// Generated by gen_luts.py -- integer tables in device memory.", "#pragma once", "#include <cstdint>", "",
           "namespace llx {"]
    for ctype, name, vals in (("uint16_t", "kDevExpI", expi), ("uint16_t", "kDevExpF", expf),
                              ("uint32_t", "kDevCurve", curve_table()), ("uint32_t", "kDevPow2", pow2_table())):
        out.append(f"static __device__ const __align__(16) {ctype} {name}[{len(vals)}] = {{")
        for i in range(0, len(vals), 8):
            out.append("    " + ", ".join(f"{v}u" for v in vals[i : i + 8]) + ",")
        out.append("};")
    out.append("}  // namespace llx")
    return "\n".join(out) + "\n"


if __name__ == "__main__":
    Path(__file__).with_name("luts_data.h").write_text(render())
    Path(__file__).with_name("device_luts.h").write_text(render_device())
