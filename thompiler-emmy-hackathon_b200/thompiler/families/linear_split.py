"""Tuned family: the fused linear product of ``thompiler.families.linear`` with K cut in two, for products
whose 256-row tiles leave most SMs without one.

A cluster of four CTAs computes one 256 x BN tile: pair q (CTAs 2 q and 2 q + 1) takes half of the K
blocks with the 2-SM MMAs of ``LinearPair``, and then owns half of the columns.  Every CTA sends its
sums of the columns that the other pair owns to the CTA with its rows there, through distributed
shared memory, into the stages that the finished product no longer needs; the owner adds them to
its own, applies the epilogue and stores.  So the long part (the MMAs of a tile) and the last (its
epilogue) are both half as long, for one exchange:

  the CTAs meet when both pairs' last MMA is done (the stages are free), send, and meet again.

512 x 4096 x 8192 bf16 on 128 SMs: 28.5 us, ``LinearPair`` with 256 x 128 tiles on as many 31.4: each
SM reads 24 KB a K block there for 256 cycles of MMAs, more than L2 delivers, where a 256 x 256
tile reads 32 KB for 512.  The exchange is bound by the SMs' network: 64 KB a CTA take 4,050 cycles,
2.1 us, as 128-byte and as 512-byte stores.  Clusters of eight (K in four) are slower everywhere:
16 of them do not fit at once.

Warps: 0 TMA, 1 MMA issuer (the pair's leader; allocates the tensor memory), 2 .. 9 the epilogue, two
to each quarter of the CTA's 128 rows, which take every other box of columns.  Every wait is
bounded, and a thread that gives one up meets the same cluster barriers as the others.
"""

from __future__ import annotations

from thompiler.families.base import TunedKernel
from thompiler.families.kit import Kit, desc_hi, elect_one, idesc_f16, tmap_address
from thompiler.families.linear import LinearPair, Product, Replay
from thompiler.families.matmul import BK, BM, STAGE_TILE
from thompiler.families.matmul_pair import PM, SMEM_LIMIT
from thompiler.lowering.types import BF16

EPILOGUE = 8                                 # warps
THREADS = 64 + 32 * EPILOGUE


class SplitPlan:
    """A tile width."""

    def __init__(self, p: Product, BN: int):
        self.BN = BN
        self.G = 2 if p.gated else 1
        self.kblocks = -(-p.K // BK)
        self.tile_cols = BN // self.G
        self.tiles_m, self.tiles_n = -(-p.M // PM), -(-p.N // self.tile_cols)
        self.ctas = self.tiles_m * self.tiles_n * 4
        self.own = self.tile_cols // 2                       # columns of C that a pair finishes
        self.box = 64 // p.c.ty.nbytes                       # columns of a store
        stage = (BM + BN // 2) * BK * 2
        # at least six: less would leave room beside this CTA for one that waits for tensor memory
        self.stages = min(8, (SMEM_LIMIT - p.static_smem - 2048) // stage)
        self.smem = self.stages * stage + 1024 + 256
        # sums from the other pair: [accumulator][column][128 rows]; the stores' staging follows
        self.exchange = self.G * self.own * BM * 4
        assert self.exchange + EPILOGUE * 2 * STAGE_TILE <= 6 * stage

    @property
    def possible(self) -> bool:
        """Two K blocks, a store's columns for each pair, and every cluster resident at once: 32 are (33 on the
        GPU measured), 34 take twice as long (256 x 8704 x 2048: 22.2 us, 256 x 8192 x 2048 12.6)."""
        return self.own >= self.box and self.kblocks >= 2 and self.stages >= 6 and self.ctas <= 128

    @classmethod
    def best(cls, p: Product) -> "SplitPlan | None":
        """The plan that the estimate takes for fastest, or None."""
        plans = [cls(p, BN) for BN in (256, 128)]
        return min((x for x in plans if x.possible), key=lambda x: x.estimate(p), default=None)

    def estimate(self, p: Product) -> float:
        """Microseconds: w from memory, or the K blocks of a pair (slower as more SMs draw on L2); then the
        launch, the exchange and the epilogue."""
        block = (0.249 if self.BN == 256 else 0.16) * (1 + 0.44 * self.ctas / 128) * (1.25, 1.05, 1.05, 1)[p.pieces]
        blocks = self.kblocks - self.kblocks // 2
        return 2.7 + 2.8 * self.BN / 256 + ((p.w.nbytes / 7.1e6) ** 4 + (blocks * block) ** 4) ** 0.25


class LinearSplit(LinearPair):
    family = "tcgen05-linear-split"

    def __init__(self, p: Product, plan: SplitPlan):
        TunedKernel.__init__(self, p.kernel)
        self.p, self.plan, self.epilogue = p, plan, p.epilogue
        self.a, self.b, self.c = p.x, p.w, p.c
        self.M, self.N, self.K, self.S, self.Ks = p.M, p.N, p.K, 1, p.K
        self.b_kmajor, self.static_smem = True, p.static_smem
        self.BN, self.HN, self.hrem, self.rem, self.parts, self.band = plan.BN, plan.BN // 2, 0, 0, 1, 0
        self.a_bytes, self.b_bytes = BM * BK * 2, self.HN * BK * 2
        self.stages, self.smem = plan.stages, plan.smem
        self.tile_cols, self.rank_cols = plan.tile_cols, p.N if p.gated else self.HN
        self.ctas = plan.ctas
        self.replay = Replay(self, p) if p.epilogue is not None else None

    def sidecar(self) -> dict:
        return dict(super().sidecar(), cluster=[4, 1, 1], block=[THREADS, 1, 1])

    def guard(self, generic: str) -> None:
        em, q = self.em, self.em.tmp("pred")
        bad = self.guard_launch(generic, THREADS, 4)
        em.ins(f"setp.ne.u32 {q}, {self.special('%nctaid.x')}, {self.ctas}")
        em.ins(f"@{q} bra {bad}")

    def emit_tuned(self) -> None:  # noqa: C901 - one kernel, written out in order
        em = self.em
        t, ins, place, lab = em.tmp, em.ins, em.place, em.label
        p, pl = self.p, self.plan
        BN, ST = self.BN, self.stages
        a_bytes, b_bytes = self.a_bytes, self.b_bytes
        mcommit = "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
        tma_ld = "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        self.pdl_trigger()
        q = t("pred")
        tid, warp, lane = self.special("%tid.x"), t("b32"), t("b32")
        ins(f"shr.u32 {warp}, {tid}, 5")
        ins(f"and.b32 {lane}, {tid}, 31")
        place_in, rank, part, first = self.special("%cluster_ctarank"), t("b32"), t("b32"), t("b32")
        ins(f"and.b32 {rank}, {place_in}, 1")
        ins(f"shr.u32 {part}, {place_in}, 1")
        ins(f"sub.u32 {first}, {place_in}, {rank}")             # the pair's leader
        base, b_st, bars = t("b32"), t("b32"), t("b32")
        ins(f"mov.u32 {base}, smem_pool")
        ins(f"add.u32 {base}, {base}, 1023")
        ins(f"and.b32 {base}, {base}, -1024")
        # shared (same offsets in all CTAs): A stages | B stages | barriers (full, empty per stage; sums
        # done) | the tensor memory's address, the set of maps.  Later the exchange and the stores' staging over the stages
        ins(f"add.u32 {b_st}, {base}, {ST * a_bytes}")
        ins(f"add.u32 {bars}, {base}, {ST * (a_bytes + b_bytes)}")
        empty_off, done_off, slot_off, sel_off = 8 * ST, 16 * ST, 16 * ST + 8, 16 * ST + 12
        # the cluster's tile and this pair's K blocks
        tm, tn, kb, ke = t("b32"), t("b32"), t("b32"), t("b32")
        cid = self.special("%clusterid.x")
        ins(f"rem.u32 {tm}, {cid}, {pl.tiles_m}")
        ins(f"div.u32 {tn}, {cid}, {pl.tiles_m}")
        ins(f"mul.lo.u32 {kb}, {part}, {pl.kblocks // 2}")
        ins(f"add.u32 {ke}, {part}, 1")
        ins(f"mul.lo.u32 {ke}, {ke}, {pl.kblocks}")
        ins(f"shr.u32 {ke}, {ke}, 1")
        self.start(bars, warp, tid, [1] * (2 * ST + 1), slot_off, sel_off, BN)
        self.pdl_wait()
        tmem, lbars, mask32, mask = t("b32"), t("b32"), t("b32"), t("b16")
        ins(f"ld.shared.u32 {tmem}, [{bars}+{slot_off}]")
        ins(f"mapa.shared::cluster.u32 {lbars}, {bars}, {first}")
        ins(f"shl.b32 {mask32}, 3, {first}")
        ins(f"cvt.u16.u32 {mask}, {mask32}")
        lead = t("pred")
        ins(f"setp.eq.u32 {lead}, {rank}, 0")
        tma, tmb, tmc = (tmap_address(em, self.tmap_set, 3, i) for i in range(3))
        errp = t("b64")
        ins(f"mov.u64 {errp}, thc_error")
        leave, out = lab("sp_leave"), lab("sp_out")
        self.check_maps(leave)
        kit = Kit(em, errp, leave)
        role_mma, role_epi = lab("sp_mma"), lab("sp_epi")
        ins(f"setp.eq.u32 {q}, {warp}, 1")
        ins(f"@{q} bra {role_mma}")
        ins(f"setp.gt.u32 {q}, {warp}, 1")
        ins(f"@{q} bra {role_epi}")

        # ---------------- producer (warp 0 of each CTA: this CTA's A rows and B half) ----------------
        is0, post = t("pred"), t("pred")
        elect_one(em, is0)
        ins(f"and.pred {post}, {is0}, {lead}")                # the leader posts both CTAs' bytes
        m0, n0, it = t("b32"), t("b32"), t("b32")
        ins(f"mul.lo.u32 {m0}, {tm}, {PM}")
        ins(f"mad.lo.u32 {m0}, {rank}, {BM}, {m0}")
        ins(f"mul.lo.u32 {n0}, {tn}, {self.tile_cols}")
        ins(f"mad.lo.u32 {n0}, {rank}, {self.rank_cols}, {n0}")
        ins(f"mov.u32 {it}, 0")
        ktop = lab("sp_load")
        place(ktop)
        stage, eb, fb, sa, sb, kc = (t("b32") for _ in range(6))
        ins(f"rem.u32 {stage}, {it}, {ST}")
        ins(f"mad.lo.u32 {eb}, {stage}, 8, {bars}")
        kit.wait(f"{eb}+{empty_off}", kit.parity(it, ST, flip=True), 0)
        ins(f"mad.lo.u32 {fb}, {stage}, 8, {lbars}")
        ins(f"mad.lo.u32 {sa}, {stage}, {a_bytes}, {base}")
        ins(f"mad.lo.u32 {sb}, {stage}, {b_bytes}, {b_st}")
        ins(f"mul.lo.u32 {kc}, {kb}, {BK}")
        ins(f"@{post} mbarrier.arrive.expect_tx.shared::cta.b64 _, [{eb}], {2 * (a_bytes + b_bytes)}")
        ins(f"@{is0} {tma_ld} [{sa}], [{tma}, {{{kc}, {m0}}}], [{fb}]")
        ins(f"@{is0} {tma_ld} [{sb}], [{tmb}, {{{kc}, {n0}}}], [{fb}]")
        ins(f"add.u32 {it}, {it}, 1")
        ins(f"add.u32 {kb}, {kb}, 1")
        ins(f"setp.lt.u32 {q}, {kb}, {ke}")
        ins(f"@{q} bra {ktop}")
        # every load is consumed by an MMA, and all CTAs meet after the last MMA
        ins(f"bra {leave}")

        # ---------------- MMA issuer (the leader's warp 1, for the pair) ----------------
        place(role_mma)
        ins(f"@!{lead} bra {leave}")
        one, hi, it2, more = t("pred"), t("b32"), t("b32"), t("pred")
        elect_one(em, one)
        ins(f"mov.u32 {hi}, {desc_hi(1024)}")
        ins(f"mov.u32 {it2}, 0")
        always = t("pred")
        ins(f"setp.eq.u32 {always}, {hi}, {hi}")
        idesc = idesc_f16(PM, BN, bf16=p.x.ty is BF16)
        mk = lab("sp_mma_k")
        place(mk)
        st2, fb2, sa2, sb2 = (t("b32") for _ in range(4))
        ins(f"rem.u32 {st2}, {it2}, {ST}")
        ins(f"mad.lo.u32 {fb2}, {st2}, 8, {bars}")
        kit.wait(fb2, kit.parity(it2, ST), 1)
        ins("tcgen05.fence::after_thread_sync")
        ins(f"mad.lo.u32 {sa2}, {st2}, {a_bytes}, {base}")
        ins(f"mad.lo.u32 {sb2}, {st2}, {b_bytes}, {b_st}")
        ad0, bd0 = kit.desc(sa2, 16, hi), kit.desc(sb2, 16, hi)
        ins(f"setp.ne.u32 {more}, {it2}, 0")                   # the first MMA overwrites the accumulators
        for k in range(BK // 16):
            ins(f"@{one} tcgen05.mma.cta_group::2.kind::f16 [{tmem}], {kit.desc_add(ad0, k * 32)}, "
                f"{kit.desc_add(bd0, k * 32)}, {idesc}, {always if k else more}")
        ins(f"@{one} {mcommit} [{fb2}+{empty_off}], {mask}")
        ins(f"add.u32 {it2}, {it2}, 1")
        ins(f"add.u32 {kb}, {kb}, 1")
        ins(f"setp.lt.u32 {q}, {kb}, {ke}")
        ins(f"@{q} bra {mk}")
        ins(f"@{one} {mcommit} [{bars}+{done_off}], {mask}")
        ins(f"bra {leave}")

        # ---------------- epilogue (warps 2 .. 9 of each CTA: its 128 rows) ----------------
        place(role_epi)
        self._epilogue(kit, tm, tn, rank, part, warp, lane, base, bars + f"+{done_off}", tmem, tmc)
        ins(f"bra {out}")

        # ---------------- the other warps, and threads that gave up a wait ----------------
        place(leave)
        for _ in range(2):
            ins("barrier.cluster.arrive.release")
            ins("barrier.cluster.wait.acquire")
        # every CTA has read its sums out of the tensor memory
        ins(f"setp.ne.u32 {q}, {warp}, 1")
        ins(f"@{q} bra {out}")
        ins("tcgen05.fence::after_thread_sync")
        ins(f"tcgen05.dealloc.cta_group::2.sync.aligned.b32 {tmem}, {BN}")
        place(out)

    def _epilogue(self, kit, tm, tn, rank, part, warp, lane, base, done, tmem, tmc) -> None:
        em = self.em
        t, ins, place, lab = em.tmp, em.ins, em.place, em.label
        p, pl = self.p, self.plan
        G, W, cw, HN = pl.G, pl.own, pl.box, self.HN
        boxes = W // cw
        turns = -(-boxes // 2)
        q = t("pred")
        quarter, side, row, taddr = t("b32"), t("b32"), t("b32"), t("b32")
        ins(f"and.b32 {quarter}, {warp}, 3")
        ins(f"sub.u32 {side}, {warp}, 2")
        ins(f"shr.u32 {side}, {side}, 2")
        ins(f"mad.lo.u32 {row}, {quarter}, 32, {lane}")        # this thread's row of the CTA's 128
        ins(f"shl.b32 {taddr}, {quarter}, 21")                 # (32 * quarter) << 16
        ins(f"add.u32 {taddr}, {taddr}, {tmem}")
        lane0 = t("pred")
        elect_one(em, lane0)
        # this warp's first box of the pair's own columns (with one box both warps of a quarter form it, the
        # first one stores it)
        mine = t("b32")
        ins(f"mul.lo.u32 {mine}, {part}, {W}")
        if boxes > 1:
            ins(f"mad.lo.u32 {mine}, {side}, {cw}, {mine}")
        self.offset = mine
        self.tile_begin(row, rank, tm, tn, "", "")
        zero = t("b32")
        ins(f"mov.u32 {zero}, 0")
        kit.wait(done, zero, 2)
        ins("tcgen05.fence::after_thread_sync")
        ins("barrier.cluster.arrive.release")                  # every pair's MMAs are done: the stages are free
        ins("barrier.cluster.wait.acquire")

        # the sums of the other pair's columns, half of them a warp, to the CTA with these rows there
        half = W // 2
        step = min(16, half)
        to, dst, src = t("b32"), t("b32"), t("b32")
        ins(f"xor.b32 {to}, {part}, 1")
        ins(f"mad.lo.u32 {dst}, {row}, 4, {base}")
        ins(f"mad.lo.u32 {dst}, {side}, {half * BM * 4}, {dst}")
        ins(f"mad.lo.u32 {src}, {to}, {W}, {taddr}")
        ins(f"mad.lo.u32 {src}, {side}, {half}, {src}")
        ins(f"mad.lo.u32 {to}, {to}, 2, {rank}")
        ins(f"mapa.shared::cluster.u32 {dst}, {dst}, {to}")
        for g in range(G):
            for c in range(0, half, step):
                v, a = em.tmps("b32", step), t("b32")
                ins(f"add.u32 {a}, {src}, {g * HN + c}")
                ins(f"tcgen05.ld.sync.aligned.32x32b.x{step}.b32 {{{', '.join(v)}}}, [{a}]")
                ins("tcgen05.wait::ld.sync.aligned")
                for i, x in enumerate(v):
                    ins(f"st.shared::cluster.b32 [{dst}+{(g * W + c + i) * BM * 4}], {x}")
        # this CTA's own
        sums = []
        for i in range(turns):
            sums.append([])
            for g in range(G):
                v, a = em.tmps("b32", cw), t("b32")
                ins(f"add.u32 {a}, {taddr}, {mine}")
                ins(f"add.u32 {a}, {a}, {g * HN + 2 * i * cw}")
                ins(f"tcgen05.ld.sync.aligned.32x32b.x{cw}.b32 {{{', '.join(v)}}}, [{a}]")
                sums[-1].append(v)
        ins("tcgen05.wait::ld.sync.aligned")
        ins("tcgen05.fence::before_thread_sync")
        ins("barrier.cluster.arrive.release")
        ins("barrier.cluster.wait.acquire")

        got, staged, sw, row0, col0 = (t("b32") for _ in range(5))
        ins(f"mad.lo.u32 {got}, {row}, 4, {base}")
        if boxes > 1:
            ins(f"mad.lo.u32 {got}, {side}, {cw * BM * 4}, {got}")
        ins(f"sub.u32 {staged}, {warp}, 2")
        ins(f"mad.lo.u32 {staged}, {staged}, {2 * STAGE_TILE}, {base}")
        ins(f"add.u32 {staged}, {staged}, {pl.exchange}")
        ins(f"shr.u32 {sw}, {lane}, 1")
        ins(f"and.b32 {sw}, {sw}, 3")
        places = []                                            # of a row's four 16-byte pieces, 64-byte swizzle
        for i in range(4):
            o = t("b32")
            ins(f"xor.b32 {o}, {sw}, {i}")
            ins(f"shl.b32 {o}, {o}, 4")
            ins(f"mad.lo.u32 {o}, {lane}, 64, {o}")
            ins(f"add.u32 {o}, {o}, {staged}")
            places.append(o)
        ins(f"mul.lo.u32 {row0}, {tm}, {PM}")
        ins(f"mad.lo.u32 {row0}, {rank}, {BM}, {row0}")
        ins(f"mad.lo.u32 {row0}, {quarter}, 32, {row0}")
        ins(f"mad.lo.u32 {col0}, {tn}, {self.tile_cols}, {mine}")
        stores = t("pred")
        ins(f"setp.eq.u32 {stores}, {side}, 0" if boxes == 1 else f"setp.ge.u32 {stores}, {side}, 0")
        ins(f"and.pred {stores}, {stores}, {lane0}")
        for i in range(turns):
            now = self.ahead if self.replay else None
            if self.replay and i + 1 < turns:
                self.ahead = self._fetch(2 * cw * (i + 1), cw)
            totals = []
            for g in range(G):
                own = em.tmps("f32", cw)
                for x, v in zip(own, sums[i][g]):
                    ins(f"mov.b32 {x}, {v}")
                for j, x in enumerate(own):
                    y = t("f32")
                    ins(f"ld.shared.f32 {y}, [{got}+{(g * W + 2 * i * cw + j) * BM * 4}]")
                    ins(f"add.rn.f32 {x}, {x}, {y}")
                totals.append(own)
            v = self._apply(totals, now, 2 * i * cw, cw) if self.replay else self._packed(totals[0])
            if i > 1:
                ins(f"@{lane0} cp.async.bulk.wait_group.read 1")
                ins("bar.warp.sync -1")
            for k in range(4):
                ins(f"st.shared.v4.b32 [{places[k]}+{i % 2 * STAGE_TILE}], {{{', '.join(v[4 * k:4 * k + 4])}}}")
            ins("fence.proxy.async.shared::cta")
            ins("bar.warp.sync -1")
            a, cc = t("b32"), t("b32")
            ins(f"add.u32 {a}, {staged}, {i % 2 * STAGE_TILE}")
            ins(f"add.u32 {cc}, {col0}, {2 * i * cw}")
            ins(f"@{stores} cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [{tmc}, {{{cc}, {row0}}}], [{a}]")
            ins(f"@{stores} cp.async.bulk.commit_group")
        ins(f"@{lane0} cp.async.bulk.wait_group 0")            # stores done before the CTA leaves
