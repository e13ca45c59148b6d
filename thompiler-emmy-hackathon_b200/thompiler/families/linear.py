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
waited for; bound by the tensor cores while K is above about a thousand: 2048 x 6144 x 4096 bf16 +
bias 68.4-69.7 us, 1,480-1,510 TFLOP/s.  ``linear_split`` holds the kernel for few tiles;
``LinearRows`` and ``LinearStream`` are for few rows; ``choose`` decides.
"""

from __future__ import annotations

from math import gcd

from thompiler import ir, schedules
from thompiler.families.base import TunedKernel
from thompiler.families.kit import (Kit, declare_tmap_ring, desc_hi, elect_one, idesc_f16, load_tmap_table,
                                    match_tmap_set)
from thompiler.families.matmul import BK, BM, EPI_WARPS, SM_COUNT, STAGE_TILE, THREADS
from thompiler.families.matmul_pair import PAIR_SLOTS, PM, SMEM_LIMIT, TcMatmulPair
from thompiler.families.tuning import TUNING
from thompiler.load import KernelInfo
from thompiler.lowering.types import BF16, F16, F32, Ty


TILE_TIMES = ((256, 1.0), (192, 0.79), (128, 0.65))      # of a pair's tile widths, of the widest's


class Product:
    """A recognised linear product: its buffers, sizes and epilogue."""

    def __init__(self, kernel: KernelInfo, gated: bool, epilogue):
        self.kernel = kernel
        self.x, self.w, self.c = (kernel.param(n) for n in ("x", "w", "linear"))
        self.M, self.K = self.x.shape
        self.N = self.c.shape[1]
        self.gated, self.epilogue = gated, epilogue
        # log2 of the 16-byte pieces that every row of x and w starts on: 3 where rows are whole 128-byte lines
        self.pieces = min(3, ((self.K * 2 // 16) & -(self.K * 2 // 16)).bit_length() - 1)
        # the generic path's slabs, where they are static arrays of their own
        self.static_smem = 0 if kernel.dynamic_smem_bytes else (3 if gated else 2) * 64 * 64 * 2

    @property
    def tile_ends(self) -> bool:
        """Does a tile's K loop end well within the second that the kernels' waits last?  2^20 blocks of the
        CTA-pair kernels, at up to 0.4 us each, take 0.4 s."""
        return self.K <= BK << 20

    def launches_in(self, cluster: int) -> bool:
        """Does meta.json's launch divide into clusters of this size?  They belong to the entry, so to every launch."""
        return self.kernel.grid[0] % cluster == 0

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
        row, col = ir.Var("row"), ir.Var("col")
        # clamped at C's own sizes an index is itself wherever the element is stored; at others it is not
        rows, cols = (row, schedules.clamped(row, p.M)), (col, schedules.clamped(col, p.N))
        if len(load.index) == 2 and load.index[0] in rows and load.index[1] in cols:
            return load.input, False, 0
        if len(load.index) == 1:
            e = load.index[0]
            if e in cols:
                return load.input, True, 0
            if isinstance(e, ir.BinaryExpr) and e.op == "+" and isinstance(e.right, ir.Literal) \
                    and e.left in cols and e.right.value % 8 == 0:
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

    @property
    def names(self) -> list[str]:
        """The buffers that are fetched."""
        return sorted({s[0] for s in self.sources})

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
    offset = None                # columns from the tile's first to those that this thread finishes
    # one compiled product serves every layer of a model.  Past the sets each call re-encodes one: 32 weights of
    # 4096 x 4096 at 512 rows, one after another, take 208 us a call with 8 sets (the other families') and 18.2
    # with 128; one weight 17.6 and 17.8
    map_sets = 128

    def __init__(self, p: Product):
        TunedKernel.__init__(self, p.kernel)
        self.p, self.epilogue = p, p.epilogue
        self.a, self.b, self.c = p.x, p.w, p.c
        self.M, self.N, self.K, self.S, self.Ks = p.M, p.N, p.K, 1, p.K
        self.b_kmajor, self.static_smem = True, p.static_smem
        _, _, self.BN, strips, self.hrem, self.tail_cols = min(self.plans(p))
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
        self.rem, self.parts = 0, 1                  # no K split: its partials would pass the epilogue twice
        self.full_tiles = self.tiles_m * self.tiles_n - self.hrem
        self.units = self.full_tiles + 2 * self.hrem
        if self.tail_cols:
            self.b_box = gcd(self.HN, self.tail_cols // 2)
        if strips >= 0:
            self.strips, self.tiles_n = strips, max(1, strips)
            self.full_tiles = self.tiles_m * strips
            self.units = self.full_tiles + self.tiles_m * -(-(p.N - strips * self.tile_cols) // self.tail_out())
        self.pairs = min(self.units, PAIR_SLOTS)
        self.ctas = 2 * self.pairs
        # tiles are walked in bands of as many rows as keep a band's x within 32 MB, so that it stays in L2 (two
        # halves of 63 MB) while w passes once a band.  TFLOP/s at the power limit, all rows / 4 / 8 / 16: 16384 x
        # 4096 x 4096 1030 / 1351 / 1335 / 1332, 8192^3 1192 / 1282 / 1318 / 1282, gated 8192 x 8192 x 4096
        # 1276 / 1300 / 1359 / 1390, 4096 x 4096 x 8192 1121 / 1133 / 1142 / 1120
        band = max(4, (32 << 20) // (PM * p.K * 2))
        self.band = band if self.tiles_m > band else 0
        self.replay = Replay(self, p) if p.epilogue is not None else None

    def tail_out(self) -> int:
        return self.tail_cols // 2 if self.p.gated else self.tail_cols

    def tail_rank_cols(self) -> int:
        return self.rank_cols if self.p.gated else self.tail_cols // 2

    @staticmethod
    def plans(p: Product) -> list[tuple]:
        """(time, work, width, whole strips of tiles or -1, tiles in halves, width of the tail's units) of each
        way to cut C, time and work in units of a 256-wide tile's: of the pair that runs most and in all.
        A last wave that would fill badly takes narrower units: two to each of its tiles, or strips of columns
        after the whole ones.  Us of as many units of 256, 192 and 128 columns, 2048 x 2304 W x 4096, W = 1 and
        3 waves: 27.7 and 75.0, 22.0 and 58.7, 18.1 and 47.0."""
        out, G = [], 2 if p.gated else 1
        rows = -(-p.M // PM)

        def busiest(full: int, units: int, cost: float) -> float:
            """Unit u runs on pair u mod PAIR_SLOTS; the first ``full`` are whole tiles."""
            whole = [-(-max(full - i, 0) // PAIR_SLOTS) for i in range(PAIR_SLOTS)]
            return max(w + cost * (-(-max(units - i, 0) // PAIR_SLOTS) - w) for i, w in enumerate(whole))

        for bn, cost in TILE_TIMES:
            if p.gated and bn != 256:
                continue
            strips = -(-p.N // (bn // G))
            tiles = rows * strips
            out.append((-(-tiles // PAIR_SLOTS) * cost, tiles * cost, bn, -1, 0, 0))
            if bn != 256 or tiles <= PAIR_SLOTS and not p.gated or not TUNING.matmul_half_tail:
                continue
            for width, cost in TILE_TIMES[1:]:
                if width // G % (128 // p.c.ty.nbytes):      # stores go in pairs of 64-byte boxes
                    continue
                rem = tiles % PAIR_SLOTS
                if width == 128 and rem and tiles > PAIR_SLOTS:
                    out.append((busiest(tiles - rem, tiles + rem, cost), tiles - rem + 2 * rem * cost, bn, -1, rem, width))
                for a in range(max(0, strips - 2 - 2 * PAIR_SLOTS // rows), strips):
                    full, tail = rows * a, rows * -(-(p.N - a * (bn // G)) // (width // G))
                    out.append((busiest(full, full + tail, cost), full + tail * cost, bn, a, 0, width))
        return out

    def estimate(self) -> float:
        """Microseconds (``choose`` says how the constants came about)."""
        waves, g = min(self.plans(self.p))[0], int(self.p.gated)
        block = 0.273 * (1 + 0.25 * self.ctas / SM_COUNT) * (1.4, 1.05, 1.05, 1)[self.p.pieces]
        later = max(waves - 1, 0)                    # whose epilogues run under the next MMAs
        return (2.27 + 1.71 * g + 2.47 * min(waves, 1) + (0.5 + 0.61 * g) * later
                + ((self.p.w.nbytes / 6.64e6) ** 4 + (waves * self.kblocks * block) ** 4) ** 0.25)

    def guard(self, generic: str) -> None:
        self.guard_launch(generic, THREADS, 2)

    def guard_launch(self, generic: str, threads: int, cluster: int) -> str:
        """The checks of a launch of ``threads`` in clusters of ``cluster``; the label to which one that cannot be
        served goes."""
        em = self.em
        declare_tmap_ring(em, 3, self.map_sets)
        em.module(".global .align 4 .u32 thc_error")
        em.module(".extern .shared .align 1024 .b8 smem_pool[]")
        em.entry_attrs.append(f".reqnctapercluster {cluster}, 1, 1")
        q, bad = em.tmp("pred"), em.label("unserved")
        self.check_aligned([self.a.name, self.b.name], 16, bad)     # in any launch: the generic path's copies too
        em.ins(f"setp.ne.u32 {q}, {self.special('%ntid.x')}, {threads}")
        em.ins(f"@{q} bra {generic}")
        em.ins(f"setp.lt.u32 {q}, {self.special('%tid.x')}, 32")
        self.table = load_tmap_table(em, [b.name for b in (self.a, self.b, self.c)], bad, self.map_sets, q)
        if self.replay:
            self.check_aligned(self.replay.names, 16, bad)
        self.refuse(bad, 4)
        return bad

    def sidecar(self) -> dict:
        names = [self.a.name, self.b.name, self.c.name] + (self.replay.names if self.replay else [])
        return dict(super().sidecar(), align=dict.fromkeys(names, 16))

    # ---- barriers, tensor memory and maps ----------------------------------------------------

    def set_up(self, bars, warp, tid, empty_off, accf_off, acce_off, slot_off, sel_off, _, p) -> None:
        """full and empty per stage, full per accumulator: one arrival; empty per accumulator: both CTAs'
        epilogue warps."""
        self.start(bars, warp, tid, [1] * (2 * self.stages + 2) + [2 * EPI_WARPS] * 2, slot_off, sel_off, self.tmem_cols)

    def start(self, bars, warp, tid, counts: list[int], slot_off: int, sel_off: int, cols: int) -> None:
        """At once: warp 0 searches the table of maps, warp 1 takes the pair's tensor memory, warp 2 initialises
        the barriers; then the cluster meets."""
        em = self.em
        t, ins, place, lab = em.tmp, em.ins, em.place, em.label
        done, search, init = lab("lp_ready"), lab("lp_search"), lab("lp_init")
        q, at = t("pred"), t("b32")
        ins(f"setp.eq.u32 {q}, {warp}, 0")
        ins(f"@{q} bra {search}")
        ins(f"setp.eq.u32 {q}, {warp}, 2")
        ins(f"@{q} bra {init}")
        ins(f"setp.ne.u32 {q}, {warp}, 1")
        ins(f"@{q} bra {done}")
        ins(f"add.u32 {at}, {bars}, {slot_off}")
        ins(f"tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [{at}], {cols}")
        ins("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned")
        ins(f"bra {done}")
        place(init)
        i, count = t("b32"), t("b32")
        ins(f"sub.u32 {i}, {tid}, 64")
        ins(f"setp.ge.u32 {q}, {i}, {len(counts)}")
        ins(f"@{q} bra {done}")
        ones = counts.count(1)                                 # these come first
        ins(f"setp.lt.u32 {q}, {i}, {ones}")
        ins(f"selp.u32 {count}, 1, {counts[-1]}, {q}")
        ins(f"mad.lo.u32 {at}, {i}, 8, {bars}")
        ins(f"mbarrier.init.shared::cta.b64 [{at}], {count}")
        ins("fence.mbarrier_init.release.cluster")
        ins("fence.proxy.async.shared::cta")
        ins(f"bra {done}")
        place(search)
        sel = match_tmap_set(em, *self.table)
        ins(f"st.shared.u32 [{bars}+{sel_off}], {sel}")
        place(done)
        ins("bar.warp.sync -1")
        ins("tcgen05.fence::before_thread_sync")
        ins("barrier.cluster.arrive.release")
        ins("barrier.cluster.wait.acquire")
        ins("tcgen05.fence::after_thread_sync")
        self.tmap_set = t("b32")
        ins(f"ld.shared.u32 {self.tmap_set}, [{bars}+{sel_off}]")

    def check_maps(self, end: str) -> None:
        """No set of maps for these buffers: record it and leave."""
        em = self.em
        q, a, bound = em.tmp("pred"), em.tmp("b64"), em.label("bound")
        em.ins(f"setp.lt.u32 {q}, {self.tmap_set}, {self.map_sets}")
        em.ins(f"@{q} bra {bound}")
        em.ins(f"mov.u64 {a}, thc_error")
        em.ins(f"atom.global.or.b32 {em.tmp('b32')}, [{a}], {1 << 4}")
        em.ins(f"bra {end}")
        em.place(bound)

    # ---- the epilogue, a box of columns at a time -----------------------------------------

    def tile_begin(self, row: str, rank: str, tm: str, tn: str, whole: str, part: str) -> None:
        if self.replay is None:
            return
        em, t, ins, p = self.em, self.em.tmp, self.em.ins, self.p
        self.row, self.col = t("b32"), t("b32")
        ins(f"mad.lo.u32 {self.row}, {tm}, {PM}, {row}")
        ins(f"mad.lo.u32 {self.row}, {rank}, {BM}, {self.row}")
        ins(f"mul.lo.u32 {self.col}, {tn}, {self.tile_cols}")
        if self.tail_cols:
            ins(f"@!{whole} mad.lo.u32 {self.col}, {part}, {self.tail_out()}, {self.col}")
        if self.offset:
            ins(f"add.u32 {self.col}, {self.col}, {self.offset}")
        self.row_ok = self.left = None
        if p.M % PM:
            self.row_ok = t("pred")
            ins(f"setp.lt.u32 {self.row_ok}, {self.row}, {p.M}")
        if p.N % self.tile_cols or self.strips is not None and (p.N - self.strips * self.tile_cols) % self.tail_out():
            self.left = t("b32")                     # columns from the tile's first one to N
            ins(f"sub.s32 {self.left}, {p.N}, {self.col}")
        self.at = {}
        for src in self.replay.sources:
            name, cols_only, first = src
            nb = p.kernel.param(name).ty.nbytes
            a, off = t("b64"), t("b64")
            ins(f"mad.wide.u32 {a}, {self.col}, {nb}, {em.buffer_reg(name)}")
            if not cols_only:
                ins(f"mul.wide.u32 {off}, {self.row}, {p.N}")
                ins(f"mad.lo.u64 {a}, {off}, {nb}, {a}")
            if first:
                ins(f"add.u64 {a}, {a}, {first * nb}")
            self.at[src] = a
        self.ahead = self._fetch(0, 64 // self.c.ty.nbytes)

    def _fetch(self, c0: int, cw: int, into: dict | None = None, when: str | None = None) -> dict:
        """Issue the loads of every source's elements c0 .. c0 + cw from the current box on, where ``when``
        holds: {source: packed registers} (``into``'s registers again, when given)."""
        em, t, ins = self.em, self.em.tmp, self.em.ins
        out = {}
        for src in self.replay.sources:
            name, cols_only, _ = src
            nb = self.p.kernel.param(name).ty.nbytes
            regs = []
            for k, c in enumerate(range(c0, c0 + cw, 16 // nb)):
                preds = [x for x in (when, None if cols_only else self.row_ok) if x]
                if self.left is not None:
                    q = t("pred")
                    ins(f"setp.gt.s32 {q}, {self.left}, {c}")
                    preds.append(q)
                pred = preds[0] if preds else None
                for x in preds[1:]:
                    both = t("pred")
                    ins(f"and.pred {both}, {pred}, {x}")
                    pred = both
                four = into[src][4 * k:4 * k + 4] if into else em.tmps("b32", 4)
                if pred is not None and not into:
                    for x in four:
                        ins(f"mov.u32 {x}, 0")
                ins(f"{f'@{pred} ' if pred else ''}ld.global.v4.b32 {{{', '.join(four)}}}, [{self.at[src]}+{c * nb}]")
                regs += four
            out[src] = regs
        return out

    def store_tile(self, cw: int, width: int, taddr: str, col0: str, free, stage) -> None:
        """The tile's boxes, two a turn of a loop: the code of a whole tile unrolled is tens of kilobytes that
        a launch of few tiles would spend its time fetching.  Each box's sources were loaded while
        the previous box was worked on."""
        em, t, ins, place, lab = self.em, self.em.tmp, self.em.ins, self.em.place, self.em.label
        turns = width // (2 * cw)
        i, ta, cc, more, last = t("b32"), t("b32"), t("b32"), t("pred"), t("pred")
        ins(f"mov.u32 {i}, 0")
        ins(f"mov.u32 {ta}, {taddr}")
        ins(f"mov.u32 {cc}, {col0}")
        top = lab("lp_box")
        place(top)
        ins(f"setp.ne.u32 {more}, {i}, {turns - 1}")
        ins(f"setp.eq.u32 {last}, {i}, {turns - 1}")
        now = self.ahead
        for b in (0, 1):
            def values(b=b):
                nonlocal now
                sums = self._sums(ta, b * cw, cw, width)
                if b == 0:
                    following = self._fetch(cw, cw)
                else:
                    following = self._fetch(2 * cw, cw, into=self.ahead, when=more)
                ins("tcgen05.wait::ld.sync.aligned")
                if b:
                    free(last)
                v = self._apply(sums, now, b * cw, cw)
                now = following
                return v
            stage(b, values, cc, b * cw)
        ins(f"add.u32 {ta}, {ta}, {2 * cw}")
        ins(f"add.u32 {cc}, {cc}, {2 * cw}")
        ins(f"add.u32 {self.col}, {self.col}, {2 * cw}")
        if self.left is not None:
            ins(f"sub.s32 {self.left}, {self.left}, {2 * cw}")
        for src, a in self.at.items():
            ins(f"add.u64 {a}, {a}, {2 * cw * self.p.kernel.param(src[0]).ty.nbytes}")
        ins(f"add.u32 {i}, {i}, 1")
        ins(f"@{more} bra {top}")

    def _sums(self, taddr: str, c0: int, cw: int, width: int) -> list[list[str]]:
        em, out = self.em, []
        for base in (c0, c0 + width) if self.p.gated else (c0,):
            v, a = em.tmps("b32", cw), em.tmp("b32")
            em.ins(f"add.u32 {a}, {taddr}, {base}")
            em.ins(f"tcgen05.ld.sync.aligned.32x32b.x{cw}.b32 {{{', '.join(v)}}}, [{a}]")
            out.append(v)
        return out

    def _apply(self, sums: list[list[str]], mine: dict, c0: int, cw: int) -> list[str]:
        """The epilogue of a box's elements, packed for the store."""
        em, t, ins = self.em, self.em.tmp, self.em.ins
        out = []
        for j in range(cw):
            z = [t("f32") for _ in sums]
            for x, v in zip(z, sums):
                ins(f"mov.b32 {x}, {v[j]}")
            col = t("b32")
            ins(f"add.u32 {col}, {self.col}, {c0 + j}")
            out.append(self.replay.element(z[0], z[1] if len(z) > 1 else None, self.row, col,
                                           lambda src, j=j: (mine[src], j)))
        return self._packed(out)

    def _packed(self, vals: list[str]) -> list[str]:
        """f32 values as the 32-bit words of C's type."""
        em, out, step = self.em, [], 4 // self.c.ty.nbytes
        for j in range(0, len(vals), step):
            out.append(em.tmp("b32"))
            em.ins(f"mov.b32 {out[-1]}, {vals[j]}" if step == 1 else
                   f"cvt.rn.{self.c.ty.ptx}x2.f32 {out[-1]}, {vals[j + 1]}, {vals[j]}")
        return out


# ---- few rows ----------------------------------------------------------------------------

ROW_SLAB = BM * BK * 2                       # one 128 x 64 slab of w
EXCHANGE_LIMIT = 64 * 1024                   # shared memory for the partial sums of a cut K
PRODUCERS = 256
MMA_WARP = PRODUCERS // 32
ROW_STEP = PRODUCERS // 8                    # rows that the producers copy a piece of at a time
OFFSET_LIMIT = 2 ** 31                       # an address' immediate offset is a signed 32-bit number


class ByElement(TunedKernel):
    """What the kernels for few rows share: a thread finishes single elements of C."""

    def __init__(self, p: Product):
        super().__init__(p.kernel)
        self.p = p
        self.replay = Replay(self, p) if p.epilogue is not None else None

    def sidecar(self) -> dict:
        return {"grid": [self.plan.ctas, 1, 1], "smem_bytes": self.plan.smem, "error_word": "thc_error",
                "align": {self.p.x.name: 16, self.p.w.name: 16}}

    def guard_launch(self, generic: str, threads: int) -> None:
        """To ``generic``: another block than ``threads``.  Refused: another grid, and, in any launch (the
        generic path copies 16 bytes at a time, too), operands off their boundary."""
        em = self.em
        em.module(".global .align 4 .u32 thc_error")
        em.module(".extern .shared .align 1024 .b8 smem_pool[]")
        q, bad = em.tmp("pred"), em.label("unserved")
        self.check_aligned([self.p.x.name, self.p.w.name], 16, bad)
        em.ins(f"setp.ne.u32 {q}, {self.special('%ntid.x')}, {threads}")
        em.ins(f"@{q} bra {generic}")
        em.ins(f"setp.ne.u32 {q}, {self.special('%nctaid.x')}, {self.plan.ctas}")
        em.ins(f"@{q} bra {bad}")
        self.refuse(bad, 4)

    def _tokens(self, x: str, m: str, n: str, left: str, inside: str | None, count: int,
                into: list | None = None) -> list:
        """Tokens x, x + 1, .. of the tile (rows m, m + 1, .. of C): [(row, stored?, sources)], with the
        sources' loads issued -- into the registers of an earlier call, when given."""
        em, t, ins, out = self.em, self.em.tmp, self.em.ins, []
        room = t("b32")
        ins(f"sub.s32 {room}, {left}, {x}")
        for j in range(count):
            mj, o, fetched = into[j] if into else (t("b32"), t("pred"), None)
            ins(f"setp.gt.s32 {o}, {room}, {j}" if inside is None else
                f"setp.gt.and.s32 {o}, {room}, {j}, {inside}")
            ins(f"add.u32 {mj}, {m}, {j}")
            out.append((mj, o, self._fetch(mj, n, o, fetched)))
        return out

    def _taken(self, ahead: list) -> list:
        """The tokens of ``ahead`` in registers of their own (the next ones are loaded over them)."""
        em, out = self.em, []
        for mj, o, fetched in ahead:
            m, p, got = em.tmp("b32"), em.tmp("pred"), dict(fetched)
            em.ins(f"mov.b32 {m}, {mj}")
            em.ins(f"mov.pred {p}, {o}")
            for src, regs in fetched.items():
                if not src[1]:
                    v = em.tmp("b32")
                    em.ins(f"mov.b32 {v}, {regs[0]}")
                    got[src] = [v]
            out.append((m, p, got))
        return out

    def _load(self, name: str, index: str, pred: str | None, into: str | None = None) -> list[str]:
        """One element of a source at a 64-bit element index, zero where ``pred`` is false."""
        em, ty = self.em, self.p.kernel.param(name).ty
        a, r = em.tmp("b64"), into or em.tmp("b32")
        em.ins(f"mad.lo.s64 {a}, {index}, {ty.nbytes}, {em.buffer_reg(name)}")
        at = f"@{pred} " if pred else ""
        em.ins(f"mov.u32 {r}, 0")
        if ty.nbytes == 4:
            em.ins(f"{at}ld.global.b32 {r}, [{a}]")
        else:
            h = em.tmp("b16")
            em.ins(f"{at}ld.global.b16 {h}, [{a}]")
            em.ins(f"{at}cvt.u32.u16 {r}, {h}")
        return [r]

    def _columns(self, n: str, inside: str | None) -> None:
        """The sources over columns, at this thread's column."""
        em = self.em
        self.cols = {}
        for src in self.replay.sources if self.replay else ():
            if src[1]:
                i = em.tmp("b64")
                em.ins(f"cvt.u64.u32 {i}, {n}")
                if src[2]:
                    em.ins(f"add.u64 {i}, {i}, {src[2]}")
                self.cols[src] = self._load(src[0], i, inside)

    def _fetch(self, m: str, n: str, ok: str, into: dict | None = None) -> dict:
        """The element sources at (m, n), and the columns' ones."""
        em, out = self.em, dict(self.cols)
        for src in self.replay.sources if self.replay else ():
            if not src[1]:
                i, c = em.tmp("b64"), em.tmp("b64")
                em.ins(f"mul.wide.u32 {i}, {m}, {self.p.N}")
                em.ins(f"cvt.u64.u32 {c}, {n}")
                em.ins(f"add.u64 {i}, {i}, {c}")
                out[src] = self._load(src[0], i, ok, into[src][0] if into else None)
        return out

    def _finish(self, sums: list[str], m: str, n: str, ok: str, fetched: dict) -> None:
        """Epilogue of one element and its store."""
        em, t, ins, c = self.em, self.em.tmp, self.em.ins, self.p.c
        vals = []
        for b in sums:
            f = t("f32")
            ins(f"mov.b32 {f}, {b}")
            vals.append(f)
        y = vals[0]
        if self.replay:
            y = self.replay.element(vals[0], vals[1] if len(vals) > 1 else None, m, n, lambda src: (fetched[src], 0))
        i, k = t("b64"), t("b64")
        ins(f"mul.wide.u32 {i}, {m}, {self.p.N}")
        ins(f"cvt.u64.u32 {k}, {n}")
        ins(f"add.u64 {i}, {i}, {k}")
        ins(f"mad.lo.s64 {i}, {i}, {c.ty.nbytes}, {em.buffer_reg(c.name)}")
        if c.ty is F32:
            ins(f"@{ok} st.global.f32 [{i}], {y}")
        else:
            h = t("b16")
            ins(f"cvt.rn.{c.ty.ptx}.f32 {h}, {y}")
            ins(f"@{ok} st.global.b16 [{i}], {h}")


class LinearRows(ByElement):
    """Few rows of x against all of w, bound by reading w once.  The roles are turned: 128 rows of w are
    the tensor cores' M side and ``BT`` rows of x (16 .. 256, exactly the batch rounded up) the N
    side, so a small batch wastes no tensor-core rows and w streams through in its own layout.

    K is cut among the ``S`` CTAs of a cluster so that every SM has w to read; each CTA sends its
    partial sums to the CTA that owns those rows of w through distributed shared memory, which adds
    them in rank order (no atomics: the same bits every time), applies the epilogue and stores.

    Eight warps copy both operands with 16-byte cp.async into the 128-byte swizzle -- no tensor maps, so
    nothing is kept for a buffer's address, and any number of weights share the kernel in captured
    graphs -- each thread's copies of a stage arriving on its mbarrier as they land; a ninth warp
    allocates the tensor memory (while the first loads are on their way), waits, fences the proxies
    and issues the MMAs.  Out-of-range rows and K are zero-filled by the copies.  Every wait is bounded."""

    family = "tcgen05-linear-rows"

    def __init__(self, p: Product, plan: "RowsPlan"):
        super().__init__(p)
        self.plan = plan

    def sidecar(self) -> dict:
        pl = self.plan
        return dict(super().sidecar(), block=[PRODUCERS + 32, 1, 1], cluster=[pl.S, 1, 1], tile=[BM, pl.BT, BK],
                    stages=pl.stages)

    def guard(self, generic: str) -> None:
        if self.plan.S > 1:
            self.em.entry_attrs.append(f".reqnctapercluster {self.plan.S}, 1, 1")
        self.guard_launch(generic, PRODUCERS + 32)

    def emit_tuned(self) -> None:  # noqa: C901 - one kernel, written out in order
        em, t, ins, place, lab = self.em, self.em.tmp, self.em.ins, self.em.place, self.em.label
        p, pl = self.p, self.plan
        S, BT, ST, G = pl.S, pl.BT, pl.stages, pl.G
        stage_bytes = pl.stage_bytes
        q = t("pred")
        tid, warp, lane = self.special("%tid.x"), t("b32"), t("b32")
        ins(f"shr.u32 {warp}, {tid}, 5")
        ins(f"and.b32 {lane}, {tid}, 31")
        base = t("b32")
        ins(f"mov.u32 {base}, smem_pool")
        ins(f"add.u32 {base}, {base}, 1023")
        ins(f"and.b32 {base}, {base}, -1024")
        # shared: stages (w slabs | x rows) | exchange | barriers (full, empty per stage; sums done; tensor
        # memory allocated) | its address
        ex, bars = t("b32"), t("b32")
        ins(f"add.u32 {ex}, {base}, {ST * stage_bytes}")
        ins(f"add.u32 {bars}, {ex}, {pl.exchange}")
        empty_off, done_off, alloc_off, slot_off = 8 * ST, 16 * ST, 16 * ST + 8, 16 * ST + 16
        # one thread a barrier: the first ST (full) expect every producer, the others one arrival
        skip, where, count = lab("lr_noinit"), t("b32"), t("b32")
        ins(f"setp.ge.u32 {q}, {tid}, {2 * ST + 2}")
        ins(f"@{q} bra {skip}")
        ins(f"mad.lo.u32 {where}, {tid}, 8, {bars}")
        ins(f"setp.lt.u32 {q}, {tid}, {ST}")
        ins(f"selp.u32 {count}, {PRODUCERS}, 1, {q}")
        ins(f"mbarrier.init.shared::cta.b64 [{where}], {count}")
        ins("fence.mbarrier_init.release.cluster")
        place(skip)
        ins("bar.sync 0")
        if S > 1:                     # met again before the first store into another CTA's shared memory
            ins("barrier.cluster.arrive.release")
        errp = t("b64")
        ins(f"mov.u64 {errp}, thc_error")
        end, fail = lab("lr_end"), lab("lr_fail")
        kit = Kit(em, errp, fail)

        # unit: the cluster's rank r holds K blocks [r kb / S, (r + 1) kb / S) of w tile tn, x tile tm
        cta, rank, unit = self.special("%ctaid.x"), t("b32"), t("b32")
        ins(f"and.b32 {rank}, {cta}, {S - 1}")
        ins(f"shr.u32 {unit}, {cta}, {S.bit_length() - 1}")
        tn, tm, n0, m0 = t("b32"), t("b32"), t("b32"), t("b32")
        ins(f"rem.u32 {tm}, {unit}, {pl.tiles_m}")
        ins(f"div.u32 {tn}, {unit}, {pl.tiles_m}")
        ins(f"mul.lo.u32 {n0}, {tn}, {BM}")
        ins(f"mul.lo.u32 {m0}, {tm}, {BT}")
        kb, nk = t("b32"), t("b32")
        ins(f"mul.lo.u32 {kb}, {rank}, {pl.kblocks}")
        ins(f"div.u32 {kb}, {kb}, {S}")
        ins(f"mad.lo.u32 {nk}, {rank}, {pl.kblocks}, {pl.kblocks}")
        ins(f"div.u32 {nk}, {nk}, {S}")
        ins(f"sub.u32 {nk}, {nk}, {kb}")                       # at least one: S <= kblocks
        role_mma = lab("lr_mma")
        ins(f"setp.eq.u32 {q}, {warp}, {MMA_WARP}")
        ins(f"@{q} bra {role_mma}")

        # ---------------- producers (warps 0..7), then the epilogue ----------------
        # the first stages of w start towards L2 while the previous kernel ends: a prefetch changes no value and
        # returns none (what that kernel may still write passes through L2)
        row, half_w, line, ok = t("b32"), t("b32"), t("b64"), t("pred")
        ins(f"and.b32 {row}, {tid}, {BM - 1}")
        ins(f"add.u32 {row}, {row}, {n0}")
        ins(f"setp.lt.u32 {ok}, {row}, {p.N}")
        ins(f"shr.u32 {half_w}, {tid}, {BM.bit_length() - 1}")
        if G == 2:
            ins(f"mad.lo.u32 {row}, {half_w}, {p.N}, {row}")
        ins(f"mul.wide.u32 {line}, {row}, {p.K * 2}")
        ins(f"add.u64 {line}, {line}, {em.buffer_reg(p.w.name)}")
        first_k = t("b64")
        ins(f"mul.wide.u32 {first_k}, {kb}, {BK * 2}")
        ins(f"add.u64 {line}, {line}, {first_k}")
        # only where a stage is mostly w (gated 16 x 8192 x 4096: 22.9 us without, 22.2 with; 128 x 4096 x 4096,
        # half of it x: 12.1 and 12.3); with one accumulator the second half of the threads takes the odd stages
        for i in range(0, ST if BT <= 32 * G else 0, 2 if G == 1 else 1):
            want, s_ = t("pred"), t("b32")
            ins(f"add.u32 {s_}, {half_w}, {i}" if G == 1 else f"mov.u32 {s_}, {i}")
            ins(f"setp.lt.and.u32 {want}, {s_}, {nk}, {ok}")
            a = t("b64")
            ins(f"mul.wide.u32 {a}, {s_}, {BK * 2}")
            ins(f"add.u64 {a}, {a}, {line}")
            ins(f"@{want} prefetch.global.L2 [{a}]")
        # thread -> 16-byte piece c of rows r0, r0 + 32, ..: a warp copies four whole 128-byte rows at a time
        self.pdl_wait()
        r0, c, soff, k8 = t("b32"), t("b32"), t("b32"), t("b32")
        ins(f"shr.u32 {r0}, {tid}, 3")
        ins(f"and.b32 {c}, {tid}, 7")
        ins(f"xor.b32 {soff}, {r0}, {c}")
        ins(f"and.b32 {soff}, {soff}, 7")
        ins(f"shl.b32 {soff}, {soff}, 4")
        ins(f"mad.lo.u32 {soff}, {r0}, 128, {soff}")
        ins(f"add.u32 {soff}, {soff}, {base}")
        ins(f"shl.b32 {k8}, {c}, 3")
        ins(f"mad.lo.u32 {k8}, {kb}, {BK}, {k8}")              # this piece's first k
        wp, xp = t("b64"), t("b64")

        def row_pointer(dst: str, first: str, buf: str) -> None:
            row, off = t("b32"), t("b64")
            ins(f"add.u32 {row}, {first}, {r0}")
            ins(f"mul.wide.u32 {off}, {row}, {p.K * 2}")
            ins(f"add.u64 {dst}, {em.buffer_reg(buf)}, {off}")
            ins(f"mul.wide.u32 {off}, {k8}, 2")
            ins(f"add.u64 {dst}, {dst}, {off}")

        row_pointer(wp, n0, p.w.name)
        row_pointer(xp, m0, p.x.name)

        def sizes(count: int, first: str, n: int, tile: int) -> list:
            """Bytes to read of each of ``count`` rows (None: always 16): 0 past the axis' end."""
            if n % tile == 0:
                return [None] * count
            out = []
            for i in range(count):
                row, z = t("b32"), t("b32")
                ins(f"add.u32 {row}, {first}, {r0}")
                ins(f"add.u32 {row}, {row}, {ROW_STEP * i}")
                ins(f"setp.lt.u32 {q}, {row}, {n}")
                ins(f"selp.u32 {z}, 16, 0, {q}")
                out.append(z)
            return out

        xrows = -(-BT // ROW_STEP)
        wsize, xsize = sizes(BM // ROW_STEP, n0, p.N, BM), sizes(xrows, m0, p.M, BT)
        half = t("pred")                                       # BT is a multiple of 16: the last step may be half a one
        ins(f"setp.lt.u32 {half}, {r0}, {BT - (xrows - 1) * ROW_STEP}")
        kit_it, st, stage_addr = t("b32"), t("b32"), t("b32")
        ins(f"mov.u32 {kit_it}, 0")
        ins(f"mov.u32 {st}, 0")
        ins(f"mov.u32 {stage_addr}, {soff}")
        ph = t("b32")
        ins(f"mov.u32 {ph}, 1")                                # parity of the empty barrier's previous phase
        ptop = lab("lr_load")
        place(ptop)
        eb = t("b32")
        ins(f"mad.lo.u32 {eb}, {st}, 8, {bars}")
        kit.wait(f"{eb}+{empty_off}", ph, 0)
        ksize = None
        if p.K % BK:
            ksize = t("b32")
            ins(f"setp.lt.u32 {q}, {k8}, {p.K}")
            ins(f"selp.u32 {ksize}, 16, 0, {q}")

        def copy(off: int, src: str, goff: int, size, hint: str = "", when: str = "") -> None:
            if size is not None and ksize is not None:
                z = t("b32")
                ins(f"and.b32 {z}, {size}, {ksize}")
            else:
                z = size if size is not None else ksize
            ins(f"{when}cp.async.cg.shared.global{hint} [{stage_addr}+{off}], [{src}+{goff}], 16{f', {z}' if z else ''}")

        for g in range(G):
            src = wp
            if g:
                src = t("b64")
                ins(f"add.u64 {src}, {wp}, {p.N * p.K * 2}")
            for i in range(BM // ROW_STEP):
                copy(g * ROW_SLAB + i * ROW_STEP * 128, src, i * ROW_STEP * p.K * 2, wsize[i], ".L2::256B")
        for i in range(xrows):
            copy(G * ROW_SLAB + i * ROW_STEP * 128, xp, i * ROW_STEP * p.K * 2, xsize[i],
                 when=f"@{half} " if i == xrows - 1 and BT % ROW_STEP else "")
        # this thread's arrival on the stage's barrier, once its copies have landed
        ins(f"cp.async.mbarrier.arrive.noinc.shared::cta.b64 [{eb}]")
        ins(f"add.u64 {wp}, {wp}, {BK * 2}")
        ins(f"add.u64 {xp}, {xp}, {BK * 2}")
        ins(f"add.u32 {k8}, {k8}, {BK}")
        ins(f"add.u32 {kit_it}, {kit_it}, 1")
        ins(f"add.u32 {st}, {st}, 1")
        ins(f"add.u32 {stage_addr}, {stage_addr}, {stage_bytes}")
        ins(f"setp.eq.u32 {q}, {st}, {ST}")
        ins(f"selp.u32 {st}, 0, {st}, {q}")
        ins(f"selp.b32 {stage_addr}, {soff}, {stage_addr}, {q}")
        flip = t("b32")
        ins(f"selp.u32 {flip}, 1, 0, {q}")
        ins(f"xor.b32 {ph}, {ph}, {flip}")
        ins(f"setp.lt.u32 {q}, {kit_it}, {nk}")
        ins(f"@{q} bra {ptop}")
        self._epilogue(kit, tid, warp, bars, done_off, alloc_off, slot_off, ex, rank, n0, m0, end)
        ins(f"bra {end}")

        # ---------------- MMA issuer (warp 8) ----------------
        place(role_mma)
        # tensor memory only once the previous kernel is done: its CTAs may share the SM and may still have to
        # allocate theirs, and this grid would keep it until that kernel ends
        self.pdl_wait()
        slot, tmem = t("b32"), t("b32")
        ins(f"add.u32 {slot}, {bars}, {slot_off}")
        ins(f"tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [{slot}], {pl.tmem_cols}")
        ins("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned")
        # for the same reason the next kernel's CTAs may come from here on, not before
        self.pdl_trigger()
        ins("bar.warp.sync -1")
        ins(f"ld.shared.u32 {tmem}, [{slot}]")
        first_lane = t("pred")
        ins(f"setp.eq.u32 {first_lane}, {lane}, 0")
        ins(f"@{first_lane} mbarrier.arrive.shared::cta.b64 _, [{bars}+{alloc_off}]")
        one = t("pred")
        elect_one(em, one)
        hi, it2, st2, par, first = t("b32"), t("b32"), t("b32"), t("b32"), t("pred")
        ins(f"mov.u32 {hi}, {desc_hi(1024)}")
        ins(f"mov.u32 {it2}, 0")
        ins(f"mov.u32 {st2}, 0")
        ins(f"mov.u32 {par}, 0")
        always = t("pred")
        ins(f"setp.eq.u32 {always}, {hi}, {hi}")
        idesc = idesc_f16(BM, BT, bf16=p.x.ty is BF16)
        mtop = lab("lr_mma_k")
        place(mtop)
        fb, sa = t("b32"), t("b32")
        ins(f"mad.lo.u32 {fb}, {st2}, 8, {bars}")
        kit.wait(fb, par, 1)
        # the copies wrote through the generic proxy, the tensor cores read through the async one
        ins("fence.proxy.async.shared::cta")
        ins("tcgen05.fence::after_thread_sync")
        ins(f"mad.lo.u32 {sa}, {st2}, {stage_bytes}, {base}")
        sx = t("b32")
        ins(f"add.u32 {sx}, {sa}, {G * ROW_SLAB}")
        ad0, bd0 = kit.desc(sa, 16, hi), kit.desc(sx, 16, hi)
        ins(f"setp.ne.u32 {first}, {it2}, 0")                  # the first block overwrites the accumulators
        for k in range(BK // 16):
            bd = kit.desc_add(bd0, k * 32)
            for g in range(G):
                ad = kit.desc_add(ad0, g * ROW_SLAB + k * 32)
                d = tmem
                if g:
                    d = t("b32")
                    ins(f"add.u32 {d}, {tmem}, {BT}")
                ins(f"@{one} tcgen05.mma.cta_group::1.kind::f16 [{d}], {ad}, {bd}, {idesc}, "
                    f"{always if k else first}")
        commit = "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64"
        ins(f"@{one} {commit} [{fb}+{empty_off}]")
        ins(f"add.u32 {it2}, {it2}, 1")
        ins(f"add.u32 {st2}, {st2}, 1")
        ins(f"setp.eq.u32 {q}, {st2}, {ST}")
        ins(f"selp.u32 {st2}, 0, {st2}, {q}")
        ins(f"selp.u32 {flip}, 1, 0, {q}")
        ins(f"xor.b32 {par}, {par}, {flip}")
        ins(f"setp.lt.u32 {q}, {it2}, {nk}")
        ins(f"@{q} bra {mtop}")
        ins(f"@{one} {commit} [{bars}+{done_off}]")
        # a thread that gave up a wait meets the same cluster barriers as the others
        place(fail)
        if S > 1:
            ins("barrier.cluster.wait.acquire")
            ins("barrier.cluster.arrive.release")
            ins("barrier.cluster.wait.acquire")

        # ---------------- common exit ----------------
        place(end)
        ins("cp.async.wait_all")
        ins("tcgen05.fence::before_thread_sync")
        ins("barrier.sync 0")
        nod = lab("lr_nodealloc")
        ins(f"setp.ne.u32 {q}, {warp}, {MMA_WARP}")
        ins(f"@{q} bra {nod}")
        ins("tcgen05.fence::after_thread_sync")
        ins(f"tcgen05.dealloc.cta_group::1.sync.aligned.b32 {tmem}, {pl.tmem_cols}")
        place(nod)

    def _read_sums(self, tmem: str, n: int) -> list[list[str]]:
        """The ``n`` columns at ``tmem`` of this thread's accumulator row(s)."""
        em, out = self.em, []
        for g in range(self.plan.G):
            v, a = em.tmps("b32", n), em.tmp("b32")
            em.ins(f"add.u32 {a}, {tmem}, {g * self.plan.BT}")
            em.ins(f"tcgen05.ld.sync.aligned.32x32b.x{n}.b32 {{{', '.join(v)}}}, [{a}]")
            out.append(v)
        em.ins("tcgen05.wait::ld.sync.aligned")
        return out

    def _epilogue(self, kit, tid, warp, bars, done_off, alloc_off, slot_off, ex, rank, n0, m0, end) -> None:
        """The sums of row n (of w) by token, to C[m0 + token, n].

        Warps w and w + 4 hold the same 32 rows of w and take alternate groups of eight tokens.  S = 1: a
        warp's loads and stores of one token are 32 consecutive columns of C.  S > 1: each rank owns
        128 / S rows; every CTA stores its sums of those rows into the owner's exchange area
        [rank][accumulator][token][row], a warp's 32 rows of a token in one store; the cluster meets, and
        the owner's threads (a row, four tokens) add the ranks' sums in order."""
        em, t, ins, place, lab = self.em, self.em.tmp, self.em.ins, self.em.place, self.em.label
        p, pl = self.p, self.plan
        S, BT, G = pl.S, pl.BT, pl.G
        q = t("pred")
        row, side, c = t("b32"), t("b32"), t("b32")            # of w's 128; which of the two warps; first token
        ins(f"and.b32 {row}, {tid}, {BM - 1}")
        ins(f"shr.u32 {side}, {warp}, 2")
        ins(f"shl.b32 {c}, {side}, 3")
        left = t("b32")                                        # tokens of this tile
        ins(f"sub.s32 {left}, {p.M}, {m0}")
        ins(f"min.s32 {left}, {left}, {BT}")
        zero, acc = t("b32"), t("b32")
        ins(f"mov.u32 {zero}, 0")

        def sums_ready() -> None:
            """Every MMA is done: ``acc`` addresses this thread's row at token c."""
            kit.wait(f"{bars}+{alloc_off}", zero, 2)
            kit.wait(f"{bars}+{done_off}", zero, 2)
            ins("tcgen05.fence::after_thread_sync")
            ins(f"ld.shared.u32 {acc}, [{bars}+{slot_off}]")
            ins(f"add.u32 {acc}, {acc}, {c}")
            lanes = t("b32")
            ins(f"and.b32 {lanes}, {warp}, 3")
            ins(f"shl.b32 {lanes}, {lanes}, 21")               # (32 * (warp mod 4)) << 16
            ins(f"add.u32 {acc}, {acc}, {lanes}")

        if S == 1:
            n, m = t("b32"), t("b32")
            ins(f"add.u32 {n}, {n0}, {row}")
            inside = None
            if p.N % BM:
                inside = t("pred")
                ins(f"setp.lt.u32 {inside}, {n}, {p.N}")
            self._columns(n, inside)
            ins(f"add.u32 {m}, {m0}, {c}")
            ahead = self._tokens(c, m, n, left, inside, 8)
            sums_ready()
            ins(f"setp.ge.s32 {q}, {c}, {left}")
            ins(f"@{q} bra {end}")
            top = lab("lr_out")
            place(top)
            sums = self._read_sums(acc, 8)
            mine = self._taken(ahead)
            ins(f"add.u32 {c}, {c}, 16")
            ins(f"add.u32 {m}, {m}, 16")
            ins(f"add.u32 {acc}, {acc}, 16")
            self._tokens(c, m, n, left, inside, 8, into=ahead)
            for j, (mj, o, fetched) in enumerate(mine):
                self._finish([v[j] for v in sums], mj, n, o, fetched)
            ins(f"setp.lt.s32 {q}, {c}, {left}")
            ins(f"@{q} bra {top}")
            return
        RS = BM // S                                           # rows of w a rank owns
        slab = BT * RS * 4                                     # bytes of one rank's sums of one accumulator
        owner, dst, dsm = t("b32"), t("b32"), t("b32")
        ins(f"shr.u32 {owner}, {row}, {RS.bit_length() - 1}")
        ins(f"and.b32 {row}, {row}, {RS - 1}")
        ins(f"mad.lo.u32 {dst}, {rank}, {G * slab}, {ex}")
        ins(f"mad.lo.u32 {dst}, {row}, 4, {dst}")
        ins(f"mad.lo.u32 {dst}, {c}, {RS * 4}, {dst}")
        ins(f"mapa.shared::cluster.u32 {dsm}, {dst}, {owner}")
        # this thread's part of the join: one of this rank's rows, tokens x .. x + 3
        n, x, m, src = t("b32"), t("b32"), t("b32"), t("b32")
        ins(f"and.b32 {n}, {tid}, {RS - 1}")
        ins(f"mad.lo.u32 {src}, {n}, 4, {ex}")
        ins(f"mad.lo.u32 {n}, {rank}, {RS}, {n}")
        ins(f"add.u32 {n}, {n}, {n0}")
        ins(f"shr.u32 {x}, {tid}, {RS.bit_length() - 1}")
        ins(f"shl.b32 {x}, {x}, 2")
        ins(f"mad.lo.u32 {src}, {x}, {RS * 4}, {src}")
        ins(f"add.u32 {m}, {m0}, {x}")
        stride = 4 * (PRODUCERS // RS)                         # tokens of a turn
        inside = None
        if p.N % BM:
            inside = t("pred")
            ins(f"setp.lt.u32 {inside}, {n}, {p.N}")
        self._columns(n, inside)
        ahead = self._tokens(x, m, n, left, inside, 4)
        sums_ready()
        ins("barrier.cluster.wait.acquire")
        send, sent, ok, room = lab("lr_send"), lab("lr_sent"), t("pred"), t("b32")
        ins(f"setp.ge.s32 {q}, {c}, {left}")
        ins(f"@{q} bra {sent}")
        place(send)
        sums = self._read_sums(acc, 8)
        ins(f"sub.s32 {room}, {left}, {c}")
        for h in range(8):
            if h:
                ins(f"setp.gt.s32 {ok}, {room}, {h}")
            for g in range(G):
                ins(f"{f'@{ok} ' if h else ''}st.shared::cluster.b32 [{dsm}+{g * slab + h * RS * 4}], {sums[g][h]}")
        ins(f"add.u32 {c}, {c}, 16")
        ins(f"add.u32 {acc}, {acc}, 16")
        ins(f"add.u32 {dsm}, {dsm}, {16 * RS * 4}")
        ins(f"setp.lt.s32 {q}, {c}, {left}")
        ins(f"@{q} bra {send}")
        place(sent)
        ins("barrier.cluster.arrive.release")
        ins("barrier.cluster.wait.acquire")
        ins(f"setp.ge.s32 {q}, {x}, {left}")
        ins(f"@{q} bra {end}")
        top = lab("lr_out")
        place(top)
        todo = self._taken(ahead)
        ins(f"add.u32 {x}, {x}, {stride}")
        ins(f"add.u32 {m}, {m}, {stride}")
        self._tokens(x, m, n, left, inside, 4, into=ahead)
        totals = []
        for g in range(G):
            total = None
            for k in range(S):
                v = em.tmps("f32", 4)
                for h, (a, (_, ok, _)) in enumerate(zip(v, todo)):
                    ins(f"mov.f32 {a}, {F32.imm(0.0)}")
                    ins(f"@{ok} ld.shared.f32 {a}, [{src}+{(k * G + g) * slab + h * RS * 4}]")
                if total is None:
                    total = v
                else:
                    for a, b in zip(total, v):
                        ins(f"add.rn.f32 {a}, {a}, {b}")
            totals.append(total)
        for j, (mj, ok, fetched) in enumerate(todo):
            bits = []
            for total in totals:
                bits.append(t("b32"))
                ins(f"mov.b32 {bits[-1]}, {total[j]}")
            self._finish(bits, mj, n, ok, fetched)
        ins(f"add.u32 {src}, {src}, {stride * RS * 4}")
        ins(f"setp.lt.s32 {q}, {x}, {left}")
        ins(f"@{q} bra {top}")


class RowsPlan:
    """Tiles and launch of ``LinearRows``: ``BT`` tokens a tile, K in ``S`` parts."""

    def __init__(self, p: Product, BT: int, S: int):
        self.BT, self.S = BT, S
        self.G = 2 if p.gated else 1
        self.kblocks = -(-p.K // BK)
        self.tiles_m, self.tiles_n = -(-p.M // BT), -(-p.N // BM)
        self.ctas = self.tiles_m * self.tiles_n * S
        self.reach = (max(BT, BM) - 1) * p.K * 2     # from a thread's first row of a tile to its last
        self.stage_bytes = self.G * ROW_SLAB + BT * BK * 2
        self.exchange = self.G * BT * BM * 4 if S > 1 else 0
        self.tmem_cols = max(32, 1 << (self.G * BT - 1).bit_length())
        # two CTAs an SM where the launch has more than one for each, or clusters so large that the SMs of a
        # processing cluster do not divide into them: of clusters of four, one CTA an SM, 33 are resident at
        # once, and a launch of 34 takes twice as long (64 x 4352 x 4096: 14.1 us, 64 x 4224 x 4096 8.3)
        half = self.ctas > (SM_COUNT if S < 4 else 128) or S == 8
        room = (SMEM_LIMIT // 2 - 1024 if half else SMEM_LIMIT) - self.exchange - 1024 - 256 - p.static_smem
        self.stages = min(12, -(-self.kblocks // S) + 1, room // self.stage_bytes)
        self.smem = self.stages * self.stage_bytes + self.exchange + 1024 + 256
        # CTAs of a cluster wait for one another while they hold tensor memory, so no two CTAs that share
        # an SM may run out of it: each takes at least its columns' share of shared memory, and more than
        # the CTA-pair kernels (all 512 columns, over 190 KB) leave
        self.smem = max(self.smem, min(SMEM_LIMIT, self.tmem_cols * 456), 36 * 1024)

    @property
    def possible(self) -> bool:
        return (self.stages >= 2 and self.S <= self.kblocks and self.exchange <= EXCHANGE_LIMIT
                and self.G * self.BT <= 512 and self.reach < OFFSET_LIMIT
                and self.ctas <= (2 * SM_COUNT if self.smem <= SMEM_LIMIT // 2 - 1024 else
                                  SM_COUNT if self.S < 4 else 128))

    @classmethod
    def best(cls, p: Product) -> "RowsPlan | None":
        """The plan that the estimate takes for fastest, or None."""
        out = []
        for tiles_m in range(1, -(-p.M // 16) + 1):
            BT = -(-(-(-p.M // tiles_m)) // 16) * 16
            if BT > 256:
                continue
            if tiles_m > 8:
                break
            for S in (1, 2, 4, 8):
                pl = cls(p, BT, S)
                if pl.possible and p.launches_in(S):
                    out.append((pl.estimate(p), S, tiles_m, pl))
        return min(out, key=lambda x: x[:3])[3] if out else None

    def estimate(self, p: Product) -> float:
        """Microseconds.  Reading w once from memory, and an SM's slabs through its copies (77 bytes a cycle,
        less where rows straddle lines -- 256 x 4096 x 2048, 2080, 2064 and 2056 take 7.8, 8.4, 9.2 and
        12.6 us, the split kernel 7.7, 7.9, 8.0 and 9.5 -- and where few stages are in flight) or tensor
        cores, overlap in part (the power mean); then the join of a cut K (large clusters wait for SMs
        that belong together) and the epilogue, by the tokens a CTA holds."""
        per_sm = -(-self.ctas // SM_COUNT)
        blocks = -(-self.kblocks // self.S)
        block = max(self.stage_bytes / 77.4 * (1.85, 1.25, 1.14, 1)[p.pieces], 1.385 * self.BT * self.G)
        if blocks > self.stages:
            block = max(block, 1142 / self.stages)
        memory, sm = p.w.nbytes / 8.28e6, per_sm * blocks * block / 1900
        tokens = self.BT * self.G / 100
        join = (0.34 + 0.89 * tokens if self.S > 1 else 0) + (1.86 if self.S == 8 and self.ctas >= 112 else 0)
        epilogue = (0.66 * tokens + 1.2 * max(0, tokens - 1.28)) * per_sm / self.S
        return 2.16 + (memory ** 1.73 + sm ** 1.73) ** (1 / 1.73) + join + epilogue


class LinearStream(ByElement):
    """A handful of rows of x (up to 24) against all of w, bound by reading w once.

    A CTA owns 16 rows of w (16 of each half when gated) and all of K; its eight warps take K in turns
    of ``U`` 32-wide chunks.  A lane loads 16 bytes of row g and of row g + 8 (g = lane / 4) at
    k = 8 (lane mod 4): taken as they lie, those registers are the A operand of two m16n8k16 MMAs whose
    k runs in another order -- the same for w and x, so the sums are the same products -- and the x
    of eight tokens, loaded by the same pattern, is their B operand.  So w goes from memory to the tensor
    cores through registers alone, with no barrier between, and a chunk's registers are loaded again
    as soon as its MMAs have read them.  The eight warps' sums meet in shared memory, added in
    warp order; a thread finishes one element at a time.

    (mma.sync, because nothing is bound by its rate here: 7 % of its cycles at 1 x 4096 x 4096, which takes
    6.1 us, 5.5 TB/s.  ``LinearRows`` takes 6.8 there: the operand barriers and the cluster's join are a
    fifth of its time, and its CTAs fill the SM's shared memory, so the next launch's cannot come early.)"""

    family = "linear-stream"

    def __init__(self, p: Product, plan: "StreamPlan"):
        super().__init__(p)
        self.plan = plan

    def sidecar(self) -> dict:
        return dict(super().sidecar(), block=[256, 1, 1])

    def guard(self, generic: str) -> None:
        self.guard_launch(generic, 256)

    def emit_tuned(self) -> None:
        em, t, ins, place, lab = self.em, self.em.tmp, self.em.ins, self.em.place, self.em.label
        p, pl = self.p, self.plan
        U, NT, G = pl.U, pl.NT, pl.G
        q = t("pred")
        self.pdl_trigger()
        tid, warp, lane, g, k8 = self.special("%tid.x"), t("b32"), t("b32"), t("b32"), t("b32")
        ins(f"shr.u32 {warp}, {tid}, 5")
        ins(f"and.b32 {lane}, {tid}, 31")
        ins(f"shr.u32 {g}, {lane}, 2")
        ins(f"and.b32 {k8}, {lane}, 3")
        n0 = t("b32")
        ins(f"shl.b32 {n0}, {self.special('%ctaid.x')}, 4")
        k = t("b32")                                           # this lane's first k of the turn
        ins(f"shl.b32 {k}, {k8}, 3")
        ins(f"mad.lo.u32 {k}, {warp}, {32 * U}, {k}")
        high = None                                            # the tile's second eight rows (N is a multiple of 8)
        if p.N % 16:
            high = t("pred")
            n8 = t("b32")
            ins(f"add.u32 {n8}, {n0}, 8")
            ins(f"setp.lt.u32 {high}, {n8}, {p.N}")

        def pointer(row: str, buf: str) -> str:
            a, o = t("b64"), t("b64")
            ins(f"mul.wide.u32 {a}, {row}, {p.K * 2}")
            ins(f"mul.wide.u32 {o}, {k}, 2")
            ins(f"add.u64 {a}, {a}, {o}")
            ins(f"add.u64 {a}, {a}, {em.buffer_reg(buf)}")
            return a

        row = t("b32")
        ins(f"add.u32 {row}, {n0}, {g}")
        wp = [pointer(row, p.w.name)]
        if G == 2:
            second = t("b64")
            ins(f"add.u64 {second}, {wp[0]}, {p.N * p.K * 2}")
            wp.append(second)
        xp, tokens = [], []
        for i in range(NT):
            tok = t("b32")
            ins(f"add.u32 {tok}, {g}, {8 * i}")
            xp.append(pointer(tok, p.x.name))
            ok = None
            if 8 * (i + 1) > p.M:
                ok = t("pred")
                ins(f"setp.lt.u32 {ok}, {tok}, {p.M}")
            tokens.append(ok)
        # the elements this thread will finish: column n, tokens tok0, tok0 + 16, ..
        n, tok0 = t("b32"), t("b32")
        ins(f"and.b32 {n}, {tid}, 15")
        ins(f"shr.u32 {tok0}, {tid}, 4")
        mine = t("b32")
        ins(f"mov.u32 {mine}, {n}")
        ins(f"add.u32 {n}, {n}, {n0}")
        inside = None
        if p.N % 16:
            inside = t("pred")
            ins(f"setp.lt.u32 {inside}, {n}, {p.N}")
        # the first turns' lines of w, four lanes a row, start towards L2 while the previous kernel ends: a
        # prefetch changes no value and returns none (what that kernel may still write passes through L2)
        line_k = t("b32")
        ins(f"shl.b32 {line_k}, {k8}, 6")
        ins(f"mad.lo.u32 {line_k}, {warp}, {32 * U}, {line_k}")
        lines = []
        for h in (0, 1):
            lr, la, lo = t("b32"), t("b64"), t("b64")
            ins(f"add.u32 {lr}, {row}, {8 * h}")
            ins(f"mul.wide.u32 {la}, {lr}, {p.K * 2}")
            ins(f"mul.wide.u32 {lo}, {line_k}, 2")
            ins(f"add.u64 {la}, {la}, {lo}")
            ins(f"add.u64 {la}, {la}, {em.buffer_reg(p.w.name)}")
            for i in range(G):
                a = la
                if i:
                    a = t("b64")
                    ins(f"add.u64 {a}, {la}, {p.N * p.K * 2}")
                lines.append((a, high if h else None))
        for turn in range(min(pl.ahead, -(-p.K // (256 * U)))):
            fits, at_k = t("pred"), t("b32")
            ins(f"add.u32 {at_k}, {line_k}, {256 * U * turn}")
            ins(f"setp.lt.u32 {fits}, {at_k}, {p.K}")
            if U < 8:                                          # a turn is fewer than four lines of a row
                ins(f"setp.lt.and.u32 {fits}, {k8}, {U // 2}, {fits}")
            for a, other in lines:
                ok = fits
                if other:
                    ok = t("pred")
                    ins(f"and.pred {ok}, {fits}, {other}")
                ins(f"@{ok} prefetch.global.L2 [{a}+{512 * U * turn}]")
        self.pdl_wait()

        w_regs = [[[em.tmps("b32", 4) for _ in range(2)] for _ in range(G)] for _ in range(U)]
        x_regs = [[em.tmps("b32", 4) for _ in range(NT)] for _ in range(U)]
        ragged = p.K % (32 * U * 8) != 0                        # some turn of some warp passes K

        def load(u: int, first: bool) -> None:
            """Chunk ``u`` of the turn that starts at k (its registers hold nothing that is still needed)."""
            fits = None
            if ragged or not first:
                fits, kk = t("pred"), t("b32")
                ins(f"add.u32 {kk}, {k}, {32 * u}")
                ins(f"setp.lt.u32 {fits}, {kk}, {p.K}")

            def both(other):
                if fits is None or other is None:
                    return fits or other
                out = t("pred")
                ins(f"and.pred {out}, {fits}, {other}")
                return out

            def one(regs, addr, off, pred, how) -> None:
                if pred is not None:
                    for x in regs:
                        ins(f"mov.u32 {x}, 0")
                ins(f"{f'@{pred} ' if pred else ''}{how}.v4.b32 {{{', '.join(regs)}}}, [{addr}+{off}]")

            for i in range(G):
                for h in (0, 1):
                    one(w_regs[u][i][h], wp[i], 64 * u + h * 8 * p.K * 2, both(high if h else None),
                        "ld.global.L1::no_allocate.L2::256B")
            for i in range(NT):
                one(x_regs[u][i], xp[i], 64 * u, both(tokens[i]), "ld.global")

        for u in range(U):
            load(u, True)
        self._columns(n, inside)
        ahead = []
        for e in range(-(-p.M // 16)):
            tok, ok = t("b32"), t("pred")
            ins(f"add.u32 {tok}, {tok0}, {16 * e}")
            ins(f"setp.lt.u32 {ok}, {tok}, {p.M}" if inside is None else
                f"setp.lt.and.u32 {ok}, {tok}, {p.M}, {inside}")
            ahead.append((tok, ok, self._fetch(tok, n, ok)))
        acc = [[em.tmps("f32", 4) for _ in range(NT)] for _ in range(G)]
        for tile in acc:
            for regs in tile:
                for x in regs:
                    ins(f"mov.f32 {x}, {F32.imm(0.0)}")
        top = lab("ls_turn")
        place(top)
        ab = p.x.ty.name
        turn = 32 * U * 8
        ins(f"add.u32 {k}, {k}, {turn}")
        for a in wp + xp:
            ins(f"add.u64 {a}, {a}, {turn * 2}")
        for u in range(U):
            for half in (0, 2):
                for i in range(G):
                    lo, hi = w_regs[u][i]
                    a = f"{{{lo[half]}, {hi[half]}, {lo[half + 1]}, {hi[half + 1]}}}"
                    for j in range(NT):
                        x = x_regs[u][j]
                        c = f"{{{', '.join(acc[i][j])}}}"
                        ins(f"mma.sync.aligned.m16n8k16.row.col.f32.{ab}.{ab}.f32 {c}, {a}, "
                            f"{{{x[half]}, {x[half + 1]}}}, {c}")
            load(u, False)
        first_k = t("b32")
        ins(f"and.b32 {first_k}, {k}, -32")                     # the turn's first k, the same in all lanes
        ins(f"setp.lt.u32 {q}, {first_k}, {p.K}")
        ins(f"@{q} bra {top}")

        # sums to shared memory: [warp][accumulator][token][16 rows, pitch 20: no two lanes share a bank]
        base, at = t("b32"), t("b32")
        ins(f"mov.u32 {base}, smem_pool")
        ins(f"mad.lo.u32 {at}, {warp}, {G * NT * 8 * 80}, {base}")
        ins(f"mad.lo.u32 {at}, {k8}, {2 * 80}, {at}")
        ins(f"mad.lo.u32 {at}, {g}, 4, {at}")
        for i in range(G):
            for j in range(NT):
                for e, x in enumerate(acc[i][j]):
                    ins(f"st.shared.f32 [{at}+{((i * NT + j) * 8 + e % 2) * 80 + (32 if e > 1 else 0)}], {x}")
        ins("bar.sync 0")
        src = t("b32")
        ins(f"mad.lo.u32 {src}, {tok0}, 80, {base}")
        ins(f"mad.lo.u32 {src}, {mine}, 4, {src}")
        for e, (tok, ok, fetched) in enumerate(ahead):
            sums = []
            for i in range(G):
                total = None
                for wv in range(8):
                    v = t("f32")
                    ins(f"mov.f32 {v}, {F32.imm(0.0)}")
                    ins(f"@{ok} ld.shared.f32 {v}, [{src}+{((wv * G + i) * NT * 8 + 16 * e) * 80}]")
                    if total is None:
                        total = v
                    else:
                        ins(f"add.rn.f32 {total}, {total}, {v}")
                bits = t("b32")
                ins(f"mov.b32 {bits}, {total}")
                sums.append(bits)
            self._finish(sums, tok, n, ok, fetched)


class StreamPlan:
    def __init__(self, p: Product):
        self.G = 2 if p.gated else 1
        self.NT = -(-p.M // 8)
        self.U = 8 if self.NT == 1 and self.G == 1 else 4
        self.ctas = -(-p.N // 16)
        # turns whose lines are asked for before the previous kernel is done.  Us with none / one / two / four:
        # 1 x 4096 x 4096 6.7 / 6.3 / 6.1 / 6.1, 4 x 1024 x 4096 4.1 / 4.0 / 3.7 / 3.6; with more CTAs than are
        # resident at once, 1 x 8192 x 8192 22.4 / 20.7 / 22.0 / 26.1
        self.ahead = 2 if self.ctas <= 2 * SM_COUNT else 1
        self.smem = 8 * self.G * self.NT * 8 * 80

    @classmethod
    def of(cls, p: Product) -> "StreamPlan | None":
        if 8 * p.K * 2 + 1024 >= OFFSET_LIMIT:     # from a lane's row of w to its second, eight further on
            return None
        return cls(p) if p.M <= 24 else None       # 32 x 4096 x 4096: 12.7 us, the rows kernel 8.0

    def estimate(self, p: Product) -> float:
        """Microseconds: w from memory, or the turns of the CTAs resident at once; past eight tokens x takes
        as many loads as w."""
        turns = -(-self.ctas // (2 * SM_COUNT)) * p.K * self.G * 0.534e-3 * (1 + 0.36 * (self.NT - 1))
        more = p.w.nbytes * (self.NT - 1) * 0.046e-6
        return 1.53 + ((p.w.nbytes / 6.46e6) ** 4 + turns ** 4) ** 0.25 + more


def choose(p: Product) -> TunedKernel | None:
    """The kernel and plan whose estimated time is least, of those whose clusters meta.json's grid divides
    into and which serve rows of this length (None: there is none).

    The estimates' forms follow what bounds each kernel; their constants are least-squares fits (of log
    time) to 1,745 timings on a B200 of every plan at M = 1 .. 1024, (N, K) from 512 x 512 to 8192 x 8192,
    plain and gated, back to back in graphs.  Over those 251 sizes the choice costs 1.0 % against the best
    plan on average and 20 % at worst; over 60 others drawn at random (M 23 .. 2400, ragged N and K) against
    the fastest kernel 1.2 % and 30 %.  Some of all sides, in us (stream / rows / split / pair):
    1 x 512 x 512 1.7 / 2.5 / - / 5.3; 1 x 4096 x 4096 6.1 / 6.8 / - / 21; 16 x 4096 x 4096 7.7 / 7.0 / - / 17;
    128 x 4096 x 4096 - / 10.3 / 12.0 / 16.5; 512 x 4096 x 8192 - / 32.1 / 28.4 / 31.4; 835 x 440 x 4048 gated
    - / 29.8 / 11.8 / 24.2; 1024 x 4096 x 4096 - / 28.8 / - / 26.3; 2048 x 4096 x 4096 - / - / - / 51."""
    plans = []
    if p.launches_in(2) and p.tile_ends:
        pair = LinearPair(p)
        plans.append((pair.estimate(), "pair", lambda: pair))
    rows, stream = RowsPlan.best(p), StreamPlan.of(p)
    if rows is not None:
        plans.append((rows.estimate(p), "rows", lambda: LinearRows(p, rows)))
    if stream is not None:
        plans.append((stream.estimate(p), "stream", lambda: LinearStream(p, stream)))
    from thompiler.families.linear_split import LinearSplit, SplitPlan
    split = SplitPlan.best(p)
    if split is not None and p.launches_in(4) and p.tile_ends:
        plans.append((split.estimate(p), "split", lambda: LinearSplit(p, split)))
    forced = [x for x in plans if x[1] == TUNING.linear_kernel]
    return min(forced or plans, key=lambda x: x[0])[2]() if plans else None


def recognise(kernel: KernelInfo):
    p = Product.read(kernel)
    return None if p is None else choose(p)
