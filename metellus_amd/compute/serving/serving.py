"""The fragment of the serving kernels: one call of a device function of
``csrc/mt_serving.h``, whose template arguments carry the sizes, strides and
launch shape that the assembly chose, and the LDS it is handed."""

from __future__ import annotations

from dataclasses import dataclass

from metellus_amd.compute.fragments import CodegenContext, TgmemAccess


@dataclass(frozen=True)
class ServingFragment:
    """``function<template args>(arguments)``; ``lds_bytes`` > 0 declares that much
    LDS as ``mt_lds`` (16-byte aligned), which ``arguments`` may name."""

    function: str
    template: tuple[int | bool, ...]
    arguments: tuple[str, ...]
    lds_bytes: int = 0
    name: str = "serving"
    kind: str = "compute"

    @property
    def tgmem_accesses(self) -> tuple[TgmemAccess, ...]:
        if not self.lds_bytes:
            return ()
        words = -(-self.lds_bytes // 4)
        return (TgmemAccess("mt_lds", "readwrite", words, (words,)),)

    def render(self, ctx: CodegenContext) -> str:
        args = ", ".join(str(v).lower() if isinstance(v, bool) else str(v) for v in self.template)
        call = f"{self.function}<{args}>({', '.join(self.arguments)});"
        if not self.lds_bytes:
            return call
        return f"alignas(16) __shared__ unsigned char mt_lds[{self.lds_bytes}];\n{call}"
