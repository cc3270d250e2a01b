"""Seeded random IR programs with the transformer operators, written as commands directly: results over operands and over
views of them, in-place updates between, branches and loops.  Every tensor but a few is [2, n, 2, 4]."""
from __future__ import annotations

import importlib

import numpy as np

adb = importlib.import_module("autodiff-ir-rust_b200")


U = 2.0 ** -24
EPS = 0.5     # a norm magnifies what a cancellation left by at most 1 / sqrt(EPS)


def tolerance(kept):
    """{id: how far a correct evaluation may be off}, or None for a program whose values grew beyond what says anything.

    Up to 60 commands of at most 16 roundings each follow one another.  A score's gradient is the difference of two sums of
    products of three values: up to 4 elements x 5 keys, 3 roundings each, of the largest magnitude cubed, whatever is left;
    four norms in a row may double that twice."""
    values = {i: np.abs(np.asarray(v.data, np.float64)) for i, v in kept.items()}
    if not all(np.isfinite(v).all() for v in values.values()):
        return None
    most = max(v.max(initial=1.0) for v in values.values())
    return None if most > 50 else {i: 60 * 16 * U * v.max(initial=0.0) + 4 * 60 * U * most ** 3 for i, v in values.items()}


def build(seed: int):
    """`prog(dev) -> {id: ValueData}`"""
    IRP = adb.ir.IRProcedure

    def prog(dev):
        rng = np.random.default_rng(seed)
        n = int(rng.integers(2, 6))
        shape = [2, n, 2, 4]
        counter = [0]

        def fresh(prefix="v"):
            counter[0] += 1
            return f"{prefix}{counter[0]}"

        def mat(block, data, dim):
            id_ = fresh("m")
            block.push(("CreateMat", np.asarray(data, np.float32).reshape(-1), list(dim), id_))
            return id_

        main = IRP("main")
        mats = [mat(main, rng.standard_normal(shape), shape) for _ in range(3)]
        scale = mat(main, 1 + 0.3 * rng.standard_normal(4), [4])
        table = mat(main, rng.uniform(0, 0.2, (2, 2)) * [[1], [1e-9]], [2, 2])
        positions = mat(main, rng.integers(0, 1000, (2, n)), [2, n])
        masks = [mat(main, rng.uniform(0, 0.5, 2), [2]), mat(main, rng.integers(-1, 2, (2, n)), [2, n]),
                 mat(main, rng.integers(0, n + 1, 2), [2]), mat(main, rng.integers(0, n + 1, 2), [2])]
        one = fresh("k")
        main.push(("CreateConstant", -1.0, one, [1]))
        anc: dict = {}     # ids that an id may be a view of (a cyclic chain of views has no meaning)

        def may_alias(res, a):
            return res == a or res in anc.get(a, ())

        def note_alias(res, a):
            new = set(anc.get(a, ())) | {a}
            anc.setdefault(res, set()).update(new)
            for s in anc.values():
                if res in s:
                    s.update(new)

        def emit(block, pool, depth):
            pool = list(pool)

            def pick():
                return pool[int(rng.integers(0, len(pool)))]

            def results(k):
                """distinct ids, new ones or in use"""
                out = []
                while len(out) < k:
                    r = fresh() if rng.random() < 0.5 else pick()
                    if r not in out:
                        out.append(r)
                return out

            def defined(ids):
                pool.extend(i for i in ids if i not in pool)

            for _ in range(int(rng.integers(3, 8))):
                kind = int(rng.integers(0, 11))
                a, b, c = pick(), pick(), pick()
                if kind == 0:
                    r = results(1)
                    block.push(("ElwAdd", a, b, r[0]))
                elif kind == 1:
                    block.push(("ElwAddEq", a, b))
                    continue
                elif kind == 2:     # heads and batch change places
                    r = results(1)
                    if may_alias(r[0], a):
                        continue
                    note_alias(r[0], a)
                    block.push(("Permute", a, [2, 1, 0, 3], r[0]))
                elif kind == 3:     # the same through two axes
                    r, w = results(1), fresh("w")
                    if may_alias(r[0], a):
                        continue
                    note_alias(w, a)
                    note_alias(r[0], w)
                    block.push(("View", a, [2 * n, 8], w))
                    block.push(("View", w, shape, r[0]))
                elif kind == 4:     # one head for both
                    r, i, w = results(1), fresh("i"), fresh("w")
                    if may_alias(r[0], a):
                        continue
                    note_alias(i, a)
                    note_alias(w, i)
                    note_alias(r[0], w)
                    block.push(("Index", a, int(rng.integers(0, 2)), 2, i))
                    block.push(("View", i, [2, n, 1, 4], w))
                    block.push(("Broadcast", w, 2, 2, r[0]))
                elif kind in (5, 6):
                    r = results(2)
                    residual = b if rng.random() < 0.5 else None
                    block.push(("RmsNorm", [a, scale, residual], r, [], [EPS]))
                elif kind == 7:
                    r, g = results(1), fresh("g")
                    block.push(("RmsNormGrad", [a, scale, b, c if rng.random() < 0.5 else None], [r[0], g], [], [EPS]))
                elif kind == 8:
                    r = results(1)
                    block.push(("Rotary", [a, table, positions if rng.random() < 0.5 else None], r,
                                [int(rng.integers(0, 2)), int(rng.integers(0, 2)), 0], [1.0]))
                else:
                    causal = int(rng.integers(0, 2))
                    m = [x if rng.random() < 0.4 else None for x in masks]
                    if not causal:
                        m[2] = None
                    reals = [0.5, float(rng.choice([0.0, 2.0]))]
                    if kind == 9:
                        r, l = results(1), fresh("l")
                        block.push(("Attention", [a, b, c] + m, [r[0], l], [causal], reals))
                    else:           # the gradient of an attention of its own, over whatever ids
                        r, o, l = results(3), fresh("o"), fresh("l")
                        block.push(("Attention", [a, b, c] + m, [o, l], [causal], reals))
                        block.push(("AttentionGrad", [a, b, c] + m + [o, l, pick()], r, [causal], reals))
                defined(r)
            if depth < 2 and rng.random() < 0.6:
                body = IRP(fresh("blk"))
                cond = fresh("c")
                if rng.random() < 0.5:
                    block.push(("CreateMat", np.asarray([rng.integers(0, 2)], np.float32), [1], cond))
                    emit(body, pool, depth + 1)
                    block.push(("If", [(cond, body)], None))
                else:
                    block.push(("CreateMat", np.asarray([rng.integers(0, 3)], np.float32), [1], cond))
                    emit(body, pool, depth + 1)
                    body.push(("ElwAddEq", cond, one))
                    block.push(("While", cond, body))
                for _ in range(2):
                    block.push(("ElwAddEq", pick(), pick()))
            return pool

        top = emit(main, mats, 0)
        keep = set(top)
        dev.execute(main, keep)
        return {i: dev.get_tensor(i) for i in sorted(keep)}

    return prog
