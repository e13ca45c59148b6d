"""Tuned family: rotary positions on packed query / key / value heads, with or without the queries'
and keys' norm (``synth.rope_package``, ``synth.qk_norm_rope_package``).

Per query or key head x[D] of a token at position p:

    n_i = x_i rsqrt(mean(x^2) + eps) w_i                       (with the norm; else n = x)
    (n_a, n_b) -> (n_a c - n_b s, n_b c + n_a s),  c, s = cos[p, i], sin[p, i]   per pair i

and values are copied.  Every element is read and written once, so memory bandwidth bounds the
large cases and the chain launch -> row load -> table load -> store the small ones.

One lane holds both elements of its pairs: V elements from the head's first half and the V that
rotate with them (16 bytes each where the sizes allow), so a rotation needs no exchange, and V
table entries serve every head of the token that the lane visits.  J = D / 2V lanes share a
head (the next power of two of lanes, the last ones idle), 32 / lanes heads a warp at a time;
the norm's sum of squares is an xor butterfly among a head's lanes, in f32.

A warp's unit is one token and up to ``rounds`` such groups of heads of one output (q, k or v:
weights and output stay the same throughout).  All of a unit's row loads are issued first, then
the position, then the tables' rows it selects and the weights: the dependent loads run under
the row loads.  A position outside the table only masks the unit's stores.
"""

from __future__ import annotations

from thompiler import ir, schedules
from thompiler.families.base import TunedKernel
from thompiler.load import KernelInfo
from thompiler.lowering.types import BF16, F16, F32, I32

SM_COUNT = 148
MAX_LANE_VALUES = 64         # f32 values of one head a lane may hold


def _pow2_at_least(n: int) -> int:
    return 1 << (n - 1).bit_length()


class RotaryHeads(TunedKernel):
    family = "rotary-heads"

    def __init__(self, kernel: KernelInfo, B, S, heads, kv, D, R, P, ty, interleaved, values, heads_first, inverse, eps):
        super().__init__(kernel)
        self.B, self.S, self.heads, self.kv, self.D, self.R, self.P = B, S, heads, kv, D, R, P
        self.ty, self.interleaved, self.values = ty, interleaved, values
        self.heads_first, self.inverse, self.eps = heads_first, inverse, eps
        self.T = B * S
        self.n = heads + kv * (2 if values else 1)
        self.V = V = schedules.heads_vector(D, R, ty.nbytes)
        self.J = D // 2 // V                                  # lanes' items in a head
        self.lanes = min(32, _pow2_at_least(self.J))
        self.items = -(-self.J // 32)                         # items a lane holds
        self.per_round = 32 // self.lanes                     # heads a warp takes at a time
        # (output, weight, first head of the row, heads)
        self.segments = [("q", "wq", 0, heads)]
        if kv:
            self.segments.append(("k", "wk", heads, kv))
        if values:
            self.segments.append(("v", None, heads + kv, kv))
        self.rounds = self._pick_rounds()
        self.units = [-(-h // (self.per_round * self.rounds)) for *_, h in self.segments]
        self.warps_needed = self.T * sum(self.units)
        self.threads = 128
        self.grid = -(-self.warps_needed // (self.threads // 32))

    def _pick_rounds(self) -> int:
        """Two rounds a unit while that leaves a warp for every scheduler, else one.  Measured at 32768 x 80
        heads of 128 bf16 with norm: one round 292 us (the coefficients' loads and the launch of twice
        the CTAs), two 225, four 239; at 3 x 1021 x 20 heads of 80: 8.7, 5.8, 6.2.  CTAs of 64, 128 and 256
        threads: 224, 225, 246 us.  A loop over further rounds in the same warp, the next one's rows loaded
        ahead, takes 249 us at its best: what it saves in table loads it loses in warps."""
        units = self.T * sum(-(-h // (2 * self.per_round)) for *_, h in self.segments)
        return 2 if self.items == 1 and units >= 4 * SM_COUNT else 1

    # ---- recognition ------------------------------------------------------------

    @classmethod
    def match(cls, kernel: KernelInfo):
        body = kernel.body
        if len(body) != 1 or not isinstance(body[0], ir.Tile) or kernel.dynamic_smem_bytes:
            return None
        qkv, pos, cos, q, k, v = (kernel.param(n) for n in ("qkv", "pos", "cos", "q", "k", "v"))
        if qkv is None or pos is None or cos is None or q is None or len(qkv.shape) != 4 or len(q.shape) != 4:
            return None
        (B, S, n, D), (P, half) = qkv.shape, cos.shape if len(cos.shape) == 2 else (0, 0)
        ty = qkv.ty
        if D % 2 or not half or ty not in (F16, BF16, F32) or B * S * n >= 2 ** 31 or pos.ty is not I32:
            return None
        eps = next((s.value.value for s in ir.walk_stmts(body) if isinstance(s, ir.Let) and s.name == "eps"), None)
        for heads_first in (False, True):
            ax = 1 if heads_first else 2
            heads, kv = q.shape[ax], k.shape[ax] if k is not None and len(k.shape) == 4 else 0
            if heads + kv * (2 if v is not None else 1) != n:
                continue
            for interleaved in (False, True):
                for inverse in (False, True):
                    args = (B, S, heads, kv, D, 2 * half, P, ty.name, interleaved, v is not None, heads_first,
                            inverse, eps)
                    if cls._shapes_ok(kernel, args) and schedules.heads_body(*args) == body[0]:
                        fam = cls(kernel, *args[:7], ty, *args[8:])
                        return fam if fam.items * 2 * fam.V <= MAX_LANE_VALUES else None
        return None

    @staticmethod
    def _shapes_ok(kernel: KernelInfo, args) -> bool:
        B, S, heads, kv, D, R, P, dt, _, values, heads_first, _, eps = args
        want = {"cos": ((P, R // 2), "f32"), "sin": ((P, R // 2), "f32"), "pos": ((B, S), "i32")}
        for name, h in (("q", heads), ("k", kv), ("v", kv if values else 0)):
            if h:
                want[name] = ((B, h, S, D) if heads_first else (B, S, h, D), dt)
        if eps is not None:
            want["wq"] = ((D,), dt)
            if kv:
                want["wk"] = ((D,), dt)
        have = {p.name: (p.shape, p.ty.name) for p in kernel.params if p.name != "qkv"}
        return have == want and R <= D

    # ---- launch ------------------------------------------------------------------

    def sidecar(self) -> dict:
        return {"grid": [self.grid, 1, 1], "block": [self.threads, 1, 1], "smem_bytes": 0,
                "error_word": "thc_error"}

    def guard(self, generic: str) -> None:
        em = self.em
        if self.eps is None and self.items == 1 and self.V <= 4:
            # room for 48 registers: left alone, the assembler keeps 32 by issuing the loads late (2 x 1777 x 16
            # heads of 96 f32: 8.6 us against 8.0).  Vectors of eight and the norm find theirs by themselves (the
            # norm's 72 capped at 64: 230 us against 225)
            em.entry_attrs += [f".maxntid {self.threads}, 1, 1", ".minnctapersm 10"]
        p = em.tmp("pred")
        em.ins(f"setp.ne.u32 {p}, {self.special('%ntid.x')}, {self.threads}")
        em.ins(f"@{p} bra {generic}")
        em.ins(f"setp.lt.u32 {p}, {self.special('%nctaid.x')}, {self.grid}")
        em.ins(f"@{p} bra {generic}")
        # every vector access aligned: V elements of the rows, up to four table entries.  (The runner refuses
        # such calls; a launch that covers the generic lowering's heads is served by it)
        bad = em.label("misaligned")
        for prm in self.k.params:
            align = 4 if prm.name == "pos" else min(16, self.V * prm.ty.nbytes)
            if align > prm.ty.nbytes:
                a = em.tmp("b64")
                em.ins(f"and.b64 {a}, {em.buffer_reg(prm.name)}, {align - 1}")
                em.ins(f"setp.ne.u64 {p}, {a}, 0")
                em.ins(f"@{p} bra {bad}")
        covered = em.label("covered")
        em.ins(f"bra {covered}")
        em.place(bad)
        em.ins(f"setp.ge.u32 {p}, {self.special('%nctaid.x')}, {-(-self.T * self.n * 32 // self.threads)}")
        em.ins(f"@{p} bra {generic}")
        short = em.label("short")
        em.ins(f"bra {short}")
        em.place(covered)
        self.refuse(short, 4)

    # ---- emission ------------------------------------------------------------------

    def _raw(self) -> int:
        """32-bit registers of V elements."""
        return max(1, self.V * self.ty.nbytes // 4)

    def _vector(self, op: str, regs: list[str], addr: str, pred: str = "") -> None:
        """Load or store V elements of the rows' type held packed in ``regs``."""
        if self.V * self.ty.nbytes == 2:
            h = self.em.tmp("b16")
            if op.startswith("ld"):
                self.em.ins(f"{pred}{op}.b16 {h}, [{addr}]")
                self.em.ins(f"{pred}cvt.u32.u16 {regs[0]}, {h}")
            else:
                self.em.ins(f"cvt.u16.u32 {h}, {regs[0]}")
                self.em.ins(f"{pred}{op}.b16 [{addr}], {h}")
            return
        n = len(regs)
        vec, body = (f".v{n}", f"{{{', '.join(regs)}}}") if n > 1 else ("", regs[0])
        if op.startswith("ld"):
            self.em.ins(f"{pred}{op}{vec}.b32 {body}, [{addr}]")
        else:
            self.em.ins(f"{pred}{op}{vec}.b32 [{addr}], {body}")

    def _unpack(self, regs: list[str]) -> list[str]:
        """V f32 values of packed elements (exact)."""
        em, out = self.em, []
        for r in regs:
            if self.ty is F32:
                f = em.tmp("f32")
                em.ins(f"mov.b32 {f}, {r}")
                out.append(f)
            elif self.ty is BF16:
                lo, hi, fl, fh = em.tmp("b32"), em.tmp("b32"), em.tmp("f32"), em.tmp("f32")
                em.ins(f"shl.b32 {lo}, {r}, 16")
                em.ins(f"and.b32 {hi}, {r}, 0xffff0000")
                em.ins(f"mov.b32 {fl}, {lo}")
                em.ins(f"mov.b32 {fh}, {hi}")
                out += [fl, fh]
            else:
                lo, hi, fl, fh = em.tmp("b16"), em.tmp("b16"), em.tmp("f32"), em.tmp("f32")
                em.ins(f"mov.b32 {{{lo}, {hi}}}, {r}")
                em.ins(f"cvt.f32.f16 {fl}, {lo}")
                em.ins(f"cvt.f32.f16 {fh}, {hi}")
                out += [fl, fh]
        return out[:self.V]

    def _pack(self, vals: list[str]) -> list[str]:
        """V f32 values rounded to the rows' type and packed."""
        em, out = self.em, []
        if self.ty is F32:
            for v in vals:
                r = em.tmp("b32")
                em.ins(f"mov.b32 {r}, {v}")
                out.append(r)
            return out
        for i in range(0, len(vals), 2):
            r = em.tmp("b32")
            hi = vals[i + 1] if i + 1 < len(vals) else F32.imm(0.0)
            em.ins(f"cvt.rn.{self.ty.ptx}x2.f32 {r}, {hi}, {vals[i]}")
            out.append(r)
        return out

    def emit_tuned(self) -> None:  # noqa: C901 - one kernel, written out in order
        em, t, ins = self.em, self.em.tmp, self.em.ins
        V, D, R, J, nb = self.V, self.D, self.R, self.J, self.ty.nbytes
        Jr = R // 2 // V
        p = t("pred")
        self.pdl_trigger()
        tid, lane, unit = self.special("%tid.x"), t("b32"), t("b32")
        ins(f"and.b32 {lane}, {tid}, 31")
        ins(f"shr.u32 {unit}, {tid}, 5")
        ins(f"mad.lo.u32 {unit}, {self.special('%ctaid.x')}, {self.threads // 32}, {unit}")
        ins(f"setp.ge.u32 {p}, {unit}, {self.warps_needed}")
        ins(f"@{p} bra {self.exit}")
        # unit -> token and the unit's place in it -> segment and first head
        upt = sum(self.units)
        token, u = t("b32"), t("b32")
        ins(f"div.u32 {token}, {unit}, {upt}")
        ins(f"rem.u32 {u}, {unit}, {upt}")
        obase, wbase = t("b64"), t("b64")
        first, seg_heads, place = t("b32"), t("b32"), t("b32")       # row's head, heads of the segment, units before
        starts = [sum(self.units[:i]) for i in range(len(self.units))]
        for i, (out, w, h0, h) in enumerate(self.segments):
            pre = ""
            if i:
                ins(f"setp.ge.u32 {p}, {u}, {starts[i]}")
                pre = f"@{p} "
            ins(f"{pre}mov.u64 {obase}, {em.buffer_reg(out)}")
            if self.eps is not None and w:
                ins(f"{pre}mov.u64 {wbase}, {em.buffer_reg(w)}")
            ins(f"{pre}mov.u32 {first}, {h0}")
            ins(f"{pre}mov.u32 {seg_heads}, {h}")
            ins(f"{pre}mov.u32 {place}, {starts[i]}")
        sub, j0 = t("b32"), t("b32")                                  # this lane's head of a round, and its first item
        ins(f"shr.u32 {sub}, {lane}, {self.lanes.bit_length() - 1}")
        ins(f"and.b32 {j0}, {lane}, {self.lanes - 1}")
        head = t("b32")
        ins(f"sub.u32 {head}, {u}, {place}")
        ins(f"mad.lo.u32 {head}, {head}, {self.per_round * self.rounds}, {sub}")

        # per item: is it one of the head's, does it rotate, byte offsets of its two vectors and its table entries
        have, turns, off0, off1, toff = [], [], [], [], []
        for i in range(self.items):
            j, a, b, c = t("b32"), t("b32"), t("b32"), t("b32")
            ins(f"add.u32 {j}, {j0}, {32 * i}")
            ok = None
            if J < 32 * (i + 1) and J != self.lanes:
                ok = t("pred")
                ins(f"setp.lt.u32 {ok}, {j}, {J}")
            rot = None
            if Jr < J:
                rot = t("pred")
                ins(f"setp.lt.u32 {rot}, {j}, {Jr}")
            step = 2 * V if self.interleaved else V
            ins(f"mul.lo.u32 {a}, {j}, {step * nb}")
            ins(f"add.u32 {b}, {a}, {(V if self.interleaved else R // 2) * nb}")
            if rot:
                a2, b2 = t("b32"), t("b32")
                ins(f"mad.lo.u32 {a2}, {j}, {2 * V * nb}, {(R - Jr * 2 * V) * nb}")
                ins(f"add.u32 {b2}, {a2}, {V * nb}")
                ins(f"selp.b32 {a}, {a}, {a2}, {rot}")
                ins(f"selp.b32 {b}, {b}, {b2}, {rot}")
            ins(f"mul.lo.u32 {c}, {j}, {V * 4}")
            have.append(ok)
            turns.append(rot)
            off0.append(a)
            off1.append(b)
            toff.append(c)

        # row pointers of the first round; the rounds' rows lie per_round heads apart
        row, xrow = t("b32"), t("b64")
        ins(f"mad.lo.u32 {row}, {token}, {self.n}, {first}")
        ins(f"add.u32 {row}, {row}, {head}")
        ins(f"mad.wide.u32 {xrow}, {row}, {D * nb}, {em.buffer_reg('qkv')}")
        orow, optr = t("b32"), t("b64")
        if self.heads_first:
            bi, si = t("b32"), t("b32")
            ins(f"div.u32 {bi}, {token}, {self.S}")
            ins(f"rem.u32 {si}, {token}, {self.S}")
            ins(f"mad.lo.u32 {orow}, {bi}, {seg_heads}, {head}")
            ins(f"mad.lo.u32 {orow}, {orow}, {self.S}, {si}")
        else:
            ins(f"mad.lo.u32 {orow}, {token}, {seg_heads}, {head}")
        ins(f"mad.wide.u32 {optr}, {orow}, {D * nb}, {obase}")
        xstep = self.per_round * D * nb
        ostep = xstep * (self.S if self.heads_first else 1)

        # from here on the warp reads and writes global data
        self.pdl_wait()
        pos, pa, inside = t("b32"), t("b64"), t("pred")               # the position; does the unit store at all?
        ins(f"mad.wide.u32 {pa}, {token}, 4, {em.buffer_reg('pos')}")
        ins(f"ld.global.u32 {pos}, [{pa}]")
        raw, live = [], []
        for r in range(self.rounds):
            ok = t("pred")
            if r:
                hr = t("b32")
                ins(f"add.u32 {hr}, {head}, {r * self.per_round}")
                ins(f"setp.lt.u32 {ok}, {hr}, {seg_heads}")
            else:
                ins(f"setp.lt.u32 {ok}, {head}, {seg_heads}")
            xr = xrow
            if r:
                xr = t("b64")
                ins(f"add.u64 {xr}, {xrow}, {r * xstep}")
            lives, raws = [], []
            for i in range(self.items):
                pi = ok
                if have[i]:
                    pi = t("pred")
                    ins(f"and.pred {pi}, {ok}, {have[i]}")
                pair = []
                for off in (off0[i], off1[i]):
                    a, w = t("b64"), t("b64")
                    ins(f"cvt.u64.u32 {w}, {off}")
                    ins(f"add.u64 {a}, {xr}, {w}")
                    regs = em.tmps("b32", self._raw())
                    for x in regs:
                        ins(f"mov.u32 {x}, 0")
                    self._vector("ld.global", regs, a, f"@{pi} ")
                    pair.append(regs)
                raws.append(pair)
                lives.append(pi)
            raw.append(raws)
            live.append(lives)

        ins(f"setp.lt.u32 {inside}, {pos}, {self.P}")                  # unsigned: negative positions lie past the table

        def store(r: int, i: int, packed) -> None:
            q = t("pred")
            ins(f"and.pred {q}, {live[r][i]}, {inside}")
            for regs, off in zip(packed, (off0[i], off1[i])):
                a, w = t("b64"), t("b64")
                ins(f"cvt.u64.u32 {w}, {off}")
                ins(f"add.u64 {a}, {optr}, {w}")
                if r:
                    ins(f"add.u64 {a}, {a}, {r * ostep}")
                self._vector("st.global", regs, a, f"@{q} ")

        if self.values:
            turned = em.label("turned")
            ins(f"setp.lt.u32 {p}, {u}, {starts[-1]}")
            ins(f"@{p} bra {turned}")
            for r in range(self.rounds):
                for i in range(self.items):
                    store(r, i, raw[r][i])
            ins(f"bra {self.exit}")
            em.place(turned)

        # the tables' entries and the weights of this lane's items, on their way while the norms are taken.  An
        # item past the rotated part has c = 1, s = 0
        tables, weights = [], []
        for i in range(self.items):
            q = inside
            for extra in (have[i], turns[i]):
                if extra:
                    q2 = t("pred")
                    ins(f"and.pred {q2}, {q}, {extra}")
                    q = q2
            tab = []
            for name, other in (("cos", 1.0), ("sin", 0.0)):
                a, w = t("b64"), t("b64")
                ins(f"mad.wide.u32 {a}, {pos}, {R // 2 * 4}, {em.buffer_reg(name)}")
                ins(f"cvt.u64.u32 {w}, {toff[i]}")
                ins(f"add.u64 {a}, {a}, {w}")
                regs = em.tmps("f32", V)
                for x in regs:
                    ins(f"mov.f32 {x}, {F32.imm(other)}")
                step = min(4, V)
                for c in range(0, V, step):
                    g = regs[c:c + step]
                    vec, body = (f".v{step}", f"{{{', '.join(g)}}}") if step > 1 else ("", g[0])
                    ins(f"@{q} ld.global{vec}.f32 {body}, [{a}{f'+{4 * c}' if c else ''}]")
                tab.append(regs)
            tables.append(tab)
            pair = []
            for off in (off0[i], off1[i]) if self.eps is not None else ():
                a, w = t("b64"), t("b64")
                ins(f"cvt.u64.u32 {w}, {off}")
                ins(f"add.u64 {a}, {wbase}, {w}")
                regs = em.tmps("b32", self._raw())
                for x in regs:
                    ins(f"mov.u32 {x}, 0")
                self._vector("ld.global", regs, a, f"@{have[i]} " if have[i] else "")
                pair.append(regs)
            weights.append(pair)

        rstd = [self._rstd(raw[r]) for r in range(self.rounds)] if self.eps is not None else []

        # the coefficients, packed two elements a register: with the weights folded in,
        # y_a = n_a (w_a c) - n_b (w_b s) and y_b = n_b (w_b c) + n_a (w_a s), n = x rstd
        coef = []
        for (cos, sin), pair in zip(tables, weights):
            ca = cb = cos
            sa = sb = sin
            if pair:
                wa, wb = self._pairs_of(*(self._unpack(x) for x in pair))
                ca, sa, cb, sb = ([self._f("mul.rn.f32", x, y) for x, y in zip(ws, tb)]
                                  for ws, tb in ((wa, cos), (wa, sin), (wb, cos), (wb, sin)))
            # the subtracted product's sine enters negated (the other one's for the inverse rotation)
            if self.inverse:
                sa = [self._f("neg.f32", x) for x in sa]
            else:
                sb = [self._f("neg.f32", x) for x in sb]
            coef.append([self._twos(x) for x in (ca, sa, cb, sb)])

        for r in range(self.rounds):
            for i in range(self.items):
                na, nb_ = (self._twos(h) for h in self._pairs_of(*(self._unpack(x) for x in raw[r][i])))
                out_a, out_b = [], []
                for m, (a, b) in enumerate(zip(na, nb_)):
                    if rstd:
                        for x in (a, b):
                            ins(f"mul.rn.f32x2 {x}, {x}, {rstd[r]}")
                    ca, sa, cb, sb = (c[m] for c in coef[i])
                    pa_, pb_, ya, yb = t("b64"), t("b64"), t("b64"), t("b64")
                    ins(f"mul.rn.f32x2 {pa_}, {a}, {ca}")
                    ins(f"mul.rn.f32x2 {pb_}, {b}, {cb}")
                    ins(f"fma.rn.f32x2 {ya}, {b}, {sb}, {pa_}")
                    ins(f"fma.rn.f32x2 {yb}, {a}, {sa}, {pb_}")
                    if turns[i]:                               # an item past the rotated part keeps its product
                        ins(f"selp.b64 {ya}, {ya}, {pa_}, {turns[i]}")
                        ins(f"selp.b64 {yb}, {yb}, {pb_}, {turns[i]}")
                    out_a.append(ya)
                    out_b.append(yb)
                v0, v1 = self._vectors_of(self._ones(out_a), self._ones(out_b))
                store(r, i, (self._pack(v0), self._pack(v1)))

    def _rstd(self, items: list) -> str:
        """rsqrt(mean(x^2) + eps) of the lane's head, twice in a 64-bit register: the squares of the lane's
        elements in two chains, then an xor butterfly among the head's lanes."""
        em, t, ins = self.em, self.em.tmp, self.em.ins
        sums = [t("b64"), t("b64")]
        for acc in sums:
            ins(f"mov.b64 {acc}, 0")
        for item in items:
            for acc, regs in zip(sums, item):
                for x in self._twos(self._unpack(regs)):
                    ins(f"fma.rn.f32x2 {acc}, {x}, {x}, {acc}")
        ins(f"add.rn.f32x2 {sums[0]}, {sums[0]}, {sums[1]}")
        lo, hi, rstd, rr = t("f32"), t("f32"), t("f32"), t("b64")
        ins(f"mov.b64 {{{lo}, {hi}}}, {sums[0]}")
        if self.V > 1:
            ins(f"add.rn.f32 {rstd}, {lo}, {hi}")
        else:                                                  # one element a register, doubled
            ins(f"mov.f32 {rstd}, {lo}")
        step = self.lanes // 2
        while step:
            o = t("f32")
            ins(f"shfl.sync.bfly.b32 {o}, {rstd}, {step}, 0x1f, 0xffffffff")
            ins(f"add.rn.f32 {rstd}, {rstd}, {o}")
            step //= 2
        ins(f"mul.rn.f32 {rstd}, {rstd}, {F32.imm(1.0 / self.D)}")
        ins(f"add.rn.f32 {rstd}, {rstd}, {F32.imm(float(self.eps))}")
        ins(f"rsqrt.approx.f32 {rstd}, {rstd}")                # relative error at most 2^-22.9
        ins(f"mov.b64 {rr}, {{{rstd}, {rstd}}}")
        return rr

    def _f(self, op: str, *args: str) -> str:
        r = self.em.tmp("f32")
        self.em.ins(f"{op} {r}, {', '.join(args)}")
        return r

    def _twos(self, vals: list[str]) -> list[str]:
        """f32 values two to a 64-bit register (an odd one doubled), for the f32x2 instructions."""
        out = []
        for m in range(0, len(vals), 2):
            out.append(self.em.tmp("b64"))
            self.em.ins(f"mov.b64 {out[-1]}, {{{vals[m]}, {vals[min(m + 1, len(vals) - 1)]}}}")
        return out

    def _ones(self, twos: list[str]) -> list[str]:
        out = []
        for x in twos:
            lo, hi = self.em.tmp("f32"), self.em.tmp("f32")
            self.em.ins(f"mov.b64 {{{lo}, {hi}}}, {x}")
            out += [lo, hi]
        return out[:self.V]

    def _pairs_of(self, v0: list, v1: list) -> tuple[list, list]:
        """The pairs' first and second elements of a lane's two vectors."""
        if not self.interleaved:
            return v0, v1
        flat = v0 + v1
        return flat[0::2], flat[1::2]

    def _vectors_of(self, a: list, b: list) -> tuple[list, list]:
        """The two vectors that hold the pairs' first and second elements ``a`` and ``b``."""
        if not self.interleaved:
            return a, b
        flat = [x for ab in zip(a, b) for x in ab]
        return flat[:self.V], flat[self.V:]


def recognise(kernel: KernelInfo):
    return RotaryHeads.match(kernel)
