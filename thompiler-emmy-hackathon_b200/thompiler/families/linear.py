"""Tuned family: the fused linear product (``synth.linear_package``),

    linear[M, N] = epilogue(x[M, K] @ w[N, K]^T),

f16 or bf16 operands, f32 sums, any M, N and K multiples of 8, and any RegStore epilogue whose
loads are a vector over the columns (a bias), an array of C's shape (a residual) or a constant:
the epilogue's own statements are replayed on the accumulators in registers, so the product,
what follows it and the one rounding are a single pass.  With a second accumulator (gated
products) the two rows of w that belong to an output column meet in the same thread.

``LinearPair``: the CTA-pair tcgen05 kernel of ``matmul_pair`` with ragged edges (TMA fills the
operands' out-of-range elements with zeros and clips the stores) and the epilogue between the
tensor memory and the store staging.  A gated tile is 256 x 128: CTA 0 of a pair holds 128 rows
of w's first half as its share of B, CTA 1 the matching 128 of the second, so accumulator
columns c and 128 + c are one output's two sums without moving a byte.  What the epilogue reads
(bias, residual) is loaded a box ahead of its use, the first box before the accumulator is
waited for; bound by the tensor cores while K is above about a thousand.
"""

from __future__ import annotations

from thompiler import ir, schedules
from thompiler.families.base import TunedKernel
from thompiler.families.matmul import BK, BM, EPI_WARPS, STAGE_TILE
from thompiler.families.matmul_pair import PAIR_SLOTS, PAIR_WIDTHS, PM, SMEM_LIMIT, TcMatmulPair
from thompiler.families.tuning import TUNING
from thompiler.load import KernelInfo
from thompiler.lowering.types import BF16, F16, F32, Ty


class Product:
    """A recognised linear product: its buffers, sizes and epilogue."""

    def __init__(self, kernel: KernelInfo, gated: bool, epilogue):
        self.kernel = kernel
        self.x, self.w, self.c = (kernel.param(n) for n in ("x", "w", "linear"))
        self.M, self.K = self.x.shape
        self.N = self.c.shape[1]
        self.gated, self.epilogue = gated, epilogue
        # the generic path's slabs, where they are static arrays of their own
        self.static_smem = 0 if kernel.dynamic_smem_bytes else (3 if gated else 2) * 64 * 64 * 2

    @classmethod
    def read(cls, kernel: KernelInfo) -> "Product | None":
        x, w, c = (kernel.param(n) for n in ("x", "w", "linear"))
        if any(p is None or len(p.shape) != 2 for p in (x, w, c)) or len(kernel.body) != 1:
            return None
        stores = [s for s in ir.walk_stmts(kernel.body) if isinstance(s, ir.RegStore)]
        if not stores or x.ty not in (F16, BF16) or w.ty is not x.ty or c.ty not in (x.ty, F32):
            return None
        gated, epi = bool(stores[0].extra_frags), stores[0].epilogue
        (M, K), N = x.shape, c.shape[1]
        if c.shape[0] != M or w.shape != (2 * N if gated else N, K) or K % 8 or N % 8:
            return None
        if epi is not None and not isinstance(epi, ir.Lambda):
            return None
        if schedules.linear_body(M, N, K, x.ty.name, gated, epi) != kernel.body[0]:
            return None
        p = cls(kernel, gated, epi)
        return p if epi is None or Replay.possible(p) else None


class Replay:
    """A RegStore epilogue's statements replayed on registers: ``sources`` are the vectors its loads
    read -- (buffer, over columns only?, first column) -- which the kernel fetches 16 bytes at a
    time, and ``element`` evaluates one element of the result."""

    def __init__(self, family, product: Product):
        self.f, self.p = family, product
        self.lam = product.epilogue
        self.sources = []
        for s in self.lam.body:
            if isinstance(s, ir.Load):
                src = self.source(product, s)
                if src is not None and src not in self.sources:
                    self.sources.append(src)

    @staticmethod
    def source(p: Product, load: ir.Load):
        """(buffer, over columns only?, first column) of a load, or None for a constant."""
        if all(isinstance(i, ir.Literal) for i in load.index):
            return None
        index = [schedules.unclamped(i) for i in load.index]
        row, col = ir.Var("row"), ir.Var("col")
        if len(index) == 2 and index == [row, col]:
            return load.input, False, 0
        if len(index) == 1:
            e = index[0]
            if e == col:
                return load.input, True, 0
            if isinstance(e, ir.BinaryExpr) and e.op == "+" and isinstance(e.right, ir.Literal) \
                    and schedules.unclamped(e.left) == col and e.right.value % 8 == 0:
                return load.input, True, e.right.value
        raise LookupError(load.input)

    @classmethod
    def possible(cls, p: Product) -> bool:
        names = [n.name if isinstance(n, ir.Var) else n for n in p.epilogue.params]
        if names not in (["z", "row", "col"], ["z", "u", "row", "col"]) or len(p.epilogue.results) != 1:
            return False
        for s in p.epilogue.body:
            if not isinstance(s, (ir.Load, ir.Assign, ir.Let, ir.Select)):
                return False
            if isinstance(s, ir.Load):
                buf = p.kernel.param(s.input)
                if len(s.names) != 1 or buf is None or buf.written or buf.ty not in (F16, BF16, F32):
                    return False
                try:
                    src = cls.source(p, s)
                except LookupError:
                    return False
                if src is not None and buf.shape != ((p.M, p.N) if not src[1] else buf.shape[:1]):
                    return False
                if src is not None and src[1] and buf.shape[0] < src[2] + p.N:
                    return False
        return True

    def check_alignment(self, generic: str) -> None:
        """Branch to ``generic`` unless every source takes 16-byte accesses."""
        em = self.f.em
        q = em.tmp("pred")
        for name in sorted({s[0] for s in self.sources}):
            a = em.tmp("b64")
            em.ins(f"and.b64 {a}, {em.buffer_reg(name)}, 15")
            em.ins(f"setp.ne.u64 {q}, {a}, 0")
            em.ins(f"@{q} bra {generic}")

    def unpacked(self, regs: list[str], i: int, ty: Ty) -> str:
        """Element ``i`` of packed ``regs`` as its load would leave it: an f32 value, or f16's b16."""
        em = self.f.em
        if ty is F32:
            r = em.tmp("f32")
            em.ins(f"mov.b32 {r}, {regs[i]}")
        elif ty is BF16:
            b, r = em.tmp("b32"), em.tmp("f32")
            em.ins(f"and.b32 {b}, {regs[i // 2]}, 0xffff0000" if i % 2 else f"shl.b32 {b}, {regs[i // 2]}, 16")
            em.ins(f"mov.b32 {r}, {b}")
        else:
            lo, hi = em.tmp("b16"), em.tmp("b16")
            em.ins(f"mov.b32 {{{lo}, {hi}}}, {regs[i // 2]}")
            r = hi if i % 2 else lo
        return r

    def element(self, z: str, u: str | None, row: str, col: str, fetched) -> str:
        """The epilogue of one element, as an f32 register; ``fetched(source)``: (packed registers,
        element's place in them)."""
        em, w = self.f.em, self.f.w

        def hook(_, load: ir.Load) -> bool:
            src = self.source(self.p, load)
            if src is None:
                return False
            ty = self.p.kernel.param(src[0]).ty
            regs, i = fetched(src)
            v = self.unpacked(regs, i, ty)
            cls = "b16" if ty is F16 else "f32"
            em.ins(f"mov.{cls} {em.value(load.names[0], cls)}, {v}")
            return True

        em.ins(f"mov.f32 {em.value('z', 'f32')}, {z}")
        if u is not None:
            em.ins(f"mov.f32 {em.value('u', 'f32')}, {u}")
        em.ins(f"mov.s32 {em.value('row', 'b32')}, {row}")
        em.ins(f"mov.s32 {em.value('col', 'b32')}, {col}")
        w.load_hook = hook
        w.body(self.lam.body)
        w.load_hook = None
        res = self.lam.results[0]
        reg = em.get(res.name if isinstance(res, ir.Var) else res)
        out = em.tmp("f32")
        em.ins(f"{'mov.f32' if em.named[reg] == 'f32' else 'cvt.f32.f16'} {out}, {reg}")
        return out


class LinearPair(TcMatmulPair):
    family = "tcgen05-linear-pair"

    def __init__(self, p: Product):
        TunedKernel.__init__(self, p.kernel)
        self.p, self.epilogue = p, p.epilogue
        self.a, self.b, self.c = p.x, p.w, p.c
        self.M, self.N, self.K, self.S, self.Ks = p.M, p.N, p.K, 1, p.K
        self.b_kmajor, self.static_smem = True, p.static_smem
        _, self.BN, self.hrem = min(self.plans(p))
        self.HN = self.BN // 2
        self.a_bytes, self.b_bytes = BM * BK * 2, self.HN * BK * 2
        stage = self.a_bytes + self.b_bytes
        self.staging = EPI_WARPS * 2 * STAGE_TILE
        room = SMEM_LIMIT - p.static_smem - 2048 - self.staging
        self.stages = max(2, min(8, room // stage))
        self.smem = self.stages * stage + self.staging + 1024 + 256
        self.tile_cols = self.HN if p.gated else self.BN
        self.rank_cols = p.N if p.gated else self.HN
        self.tiles_m, self.tiles_n = -(-p.M // PM), -(-p.N // self.tile_cols)
        self.kblocks = -(-p.K // BK)
        self.tiles = self.tiles_m * self.tiles_n
        self.rem, self.parts = 0, 1                  # no K split: its partials would pass the epilogue twice
        self.full_tiles = self.tiles - self.hrem
        self.units = self.full_tiles + 2 * self.hrem
        self.pairs = min(self.units, PAIR_SLOTS)
        self.ctas = 2 * self.pairs
        self.replay = Replay(self, p) if p.epilogue is not None else None

    @staticmethod
    def plans(p: Product) -> list[tuple[float, int, int]]:
        """(waves of a 256-wide tile's time, width, halved tiles) of each tile width: the tiles a
        pair runs in a row, each as long as its width at that width's measured efficiency; a last
        wave whose tiles halved fit one wave runs as halves, which take 0.7 of a whole."""
        out = []
        for bn, pref in PAIR_WIDTHS:
            if p.gated and bn != 256:
                continue
            tiles = -(-p.M // PM) * -(-p.N // (bn // 2 if p.gated else bn))
            waves, rem = divmod(tiles, PAIR_SLOTS)
            half = waves and rem and 2 * rem <= PAIR_SLOTS and bn == 256 and not p.gated and TUNING.matmul_half_tail
            time = waves + (0 if not rem else 0.7 if half else 1)
            out.append((time * bn / 256 / pref, bn, rem if half else 0))
        return out

    def guard(self, generic: str) -> None:
        super().guard(generic)
        if self.replay:
            self.replay.check_alignment(generic)

    # ---- the epilogue, a box of columns at a time -----------------------------------------

    def tile_begin(self, row: str, rank: str, tm: str, tn: str, whole: str, part: str) -> None:
        if self.replay is None:
            return
        em, t, ins, p = self.em, self.em.tmp, self.em.ins, self.p
        self.row, self.col = t("b32"), t("b32")
        ins(f"mad.lo.u32 {self.row}, {tm}, {PM}, {row}")
        ins(f"mad.lo.u32 {self.row}, {rank}, {BM}, {self.row}")
        ins(f"mul.lo.u32 {self.col}, {tn}, {self.tile_cols}")
        if self.hrem:
            ins(f"@!{whole} mad.lo.u32 {self.col}, {part}, {self.BN // 2}, {self.col}")
        self.row_ok = self.left = None
        if p.M % PM:
            self.row_ok = t("pred")
            ins(f"setp.lt.u32 {self.row_ok}, {self.row}, {p.M}")
        if p.N % self.tile_cols:
            self.left = t("b32")                     # columns from the tile's first one to N
            ins(f"sub.s32 {self.left}, {p.N}, {self.col}")
        self.at = {}
        for src in self.replay.sources:
            name, cols_only, first = src
            nb = p.kernel.param(name).ty.nbytes
            a, off = t("b64"), t("b64")
            ins(f"mad.wide.u32 {a}, {self.col}, {nb}, {em.buffer_reg(name)}")
            if not cols_only:
                ins(f"mul.wide.u32 {off}, {self.row}, {p.N * nb}")
                ins(f"add.u64 {a}, {a}, {off}")
            if first:
                ins(f"add.u64 {a}, {a}, {first * nb}")
            self.at[src] = a
        cw = 64 // self.c.ty.nbytes
        self.first = self._fetch(0, cw)
        self.ahead = {}

    def _fetch(self, c0: int, cw: int) -> dict:
        """Issue the loads of every source's elements c0 .. c0 + cw: {source: packed registers}."""
        em, t, ins = self.em, self.em.tmp, self.em.ins
        out = {}
        for src in self.replay.sources:
            name, cols_only, _ = src
            nb = self.p.kernel.param(name).ty.nbytes
            regs = []
            for c in range(c0, c0 + cw, 16 // nb):
                pred = None if cols_only else self.row_ok
                if self.left is not None:
                    q = t("pred")
                    ins(f"setp.gt.s32 {q}, {self.left}, {c}" if pred is None else
                        f"setp.gt.and.s32 {q}, {self.left}, {c}, {pred}")
                    pred = q
                four = em.tmps("b32", 4)
                if pred is not None:
                    for r in four:
                        ins(f"mov.u32 {r}, 0")
                ins(f"{f'@{pred} ' if pred else ''}ld.global.nc.v4.b32 {{{', '.join(four)}}}, [{self.at[src]}+{c * nb}]")
                regs += four
            out[src] = regs
        return out

    def box(self, c0: int, cw: int, width: int, taddr: str) -> list[str]:
        em, t, ins = self.em, self.em.tmp, self.em.ins
        if c0 == 0:
            self.ahead = {0: self.first}
        mine = self.ahead.pop(c0)
        sums = []
        for base in (c0, c0 + self.HN) if self.p.gated else (c0,):
            v = em.tmps("b32", cw)
            a = t("b32")
            ins(f"add.u32 {a}, {taddr}, {base}")
            ins(f"tcgen05.ld.sync.aligned.32x32b.x{cw}.b32 {{{', '.join(v)}}}, [{a}]")
            sums.append(v)
        if c0 + cw < width:
            self.ahead[c0 + cw] = self._fetch(c0 + cw, cw)
        ins("tcgen05.wait::ld.sync.aligned")
        out = []
        for j in range(cw):
            z = [t("f32") for _ in sums]
            for r, v in zip(z, sums):
                ins(f"mov.b32 {r}, {v[j]}")
            col = t("b32")
            ins(f"add.u32 {col}, {self.col}, {c0 + j}")
            out.append(self.replay.element(z[0], z[1] if len(z) > 1 else None, self.row, col,
                                           lambda src, j=j: (mine[src], j)))
        packed = []
        step = 4 // self.c.ty.nbytes
        for j in range(0, cw, step):
            r = t("b32")
            ins(f"mov.b32 {r}, {out[j]}" if step == 1 else f"cvt.rn.{self.c.ty.ptx}x2.f32 {r}, {out[j + 1]}, {out[j]}")
            packed.append(r)
        return packed


def recognise(kernel: KernelInfo):
    p = Product.read(kernel)
    if p is None:
        return None
    if p.M > 128:
        return LinearPair(p)
    return None
