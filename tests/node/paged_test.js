'use strict'
/*
 * The paged cache's calls through the N-API addon and HipGpu (CommonJS, Node
 * 12). Usage:
 *   node paged_test.js cpu    (no GPU: scratch sizes, refused arguments)
 *   node paged_test.js gpu    (two sequences prepared, attended and evicted in
 *                              pages, against the contiguous cache's calls)
 * Assertions fail the process; a JSON summary goes to stdout.
 */
const assert = require('assert')
const path = require('path')

const hip = require(path.join(__dirname, '..', '..', 'webgllm_amd', 'node', 'index.js'))

const shape = { heads: 4, kvHeads: 2, headDim: 64 }
const HD = 64
const QD = 4 * HD
const KVD = 2 * HD

function invalid (fn, text) {
  assert.throws(fn, (e) => (e instanceof hip.GpuError || e.name === 'GpuError') && e.code === 'WG_ERR_INVALID' && (!text || e.message.includes(text)))
}

function cpu () {
  const A = hip.addon
  const sizes = { pages: 9, pageSize: 16, ldTable: 4, sequences: 2 }
  const long = { pages: 9000, pageSize: 16, ldTable: 4000, sequences: 2 }
  invalid(() => A.pagedEvictScratchBytes(Object.assign({}, sizes, { pages: 0 })))
  invalid(() => A.pagedEvictScratchBytes(Object.assign({}, sizes, { pageSize: 1 << 30 })))
  invalid(() => A.pagedPrefillScratchBytes(sizes, { heads: 4, kvHeads: 0, headDim: 64 }, 3))
  assert.throws(() => A.pagedDecodeScratchBytes(null, shape, 0), TypeError)
  assert.throws(() => A.pagedDecodeScratchBytes(Object.assign({}, sizes, { sequences: 'two' }), shape, 0), TypeError)
  for (const name of ['pagedHeadPrep', 'pagedAttnDecode', 'pagedAttnPrefill', 'pagedEvict']) assert.throws(() => A[name]({}), TypeError)
  return {
    decode: [sizes, long].map((c) => A.pagedDecodeScratchBytes(c, shape, 0)),
    weights: [sizes, long].map((c) => A.pagedDecodeScratchBytes(c, shape, 1)),
    prefill: [sizes, long].map((c) => A.pagedPrefillScratchBytes(c, shape, 5)),
    evict: [sizes, long].map((c) => A.pagedEvictScratchBytes(c))
  }
}

/** Half bits to a number. */
function half (h) {
  const e = (h >> 10) & 31
  const f = h & 1023
  const v = e === 0 ? f * 2 ** -24 : e === 31 ? (f ? NaN : Infinity) : (1 + f / 1024) * 2 ** (e - 15)
  return h & 0x8000 ? -v : v
}

function gpu () {
  const { GL } = hip
  const g = new hip.HipGpu(0)
  const bytes = (n) => g.texture(GL.R8UI, n, 1, { format: 0, type: 0, pixels: new Uint8Array(n) })
  const up = (a) => g.texture(GL.R8UI, a.byteLength, 1, { format: 0, type: 0, pixels: a })
  const raw = (t, T) => new T(g.readBytes(t, 0, t.bytes))
  let seed = 1
  const rnd = () => { // (uniform, variance 1)
    seed = (Math.imul(seed, 1103515245) + 12345) >>> 0
    return ((seed >>> 8) / (1 << 24) - 0.5) * Math.sqrt(12)
  }
  const lens = [37, 20]
  const start = [0, 37, 57]
  const M = 57
  const ropeRows = 1024 + 1
  const rope = new Float32Array(ropeRows * HD)
  for (let r = 0; r < ropeRows; r++) {
    for (let i = 0; i < HD / 2; i++) {
      const a = (r < 1024 ? r : (r - 1024) * 1024) * Math.pow(1e4, -2 * i / HD)
      rope[r * HD + i] = Math.cos(a)
      rope[r * HD + HD / 2 + i] = Math.sin(a)
    }
  }
  const tRope = up(rope)
  const qkv = up(Float32Array.from({ length: M * (QD + 2 * KVD) }, rnd))
  const table = [[7, 2, 5, -1], [0, 4, -1, -1]]
  const cache = {
    k: bytes(9 * 16 * KVD * 2), v: bytes(9 * 16 * KVD * 2), pages: 9, pageSize: 16, ldTable: 4, sequences: 2,
    table: up(Int32Array.from([].concat(...table))), lens: up(Int32Array.from(lens))
  }
  const rowStart = up(Int32Array.from(start))
  // the preparation: bit for bit the contiguous call's queries, keys and values
  const q = bytes(M * QD * 4)
  g.ops.pagedHeadPrep(qkv, M, shape, null, null, tRope, ropeRows, null, cache, rowStart, q)
  const q2 = bytes(M * QD * 4)
  const pos0 = bytes(4)
  const own = lens.map((n, b) => {
    const kv = [bytes(n * KVD * 2), bytes(n * KVD * 2)]
    g.ops.headPrep(g.view(qkv, start[b] * (QD + 2 * KVD) * 4), n, shape, null, null, tRope, ropeRows, pos0,
      g.view(q2, start[b] * QD * 4), kv[0], kv[1], n)
    return kv
  })
  assert.deepStrictEqual(raw(q, Uint32Array), raw(q2, Uint32Array))
  const rowsOf = (pool, tab, n) => {
    const out = []
    for (let i = 0; i < n; i++) {
      const at = (tab[i >> 4] * 16 + (i & 15)) * KVD
      out.push(...pool.subarray(at, at + KVD))
    }
    return out
  }
  for (const [i, pool] of [cache.k, cache.v].entries()) {
    const p = raw(pool, Uint16Array)
    lens.forEach((n, b) => assert.deepStrictEqual(rowsOf(p, table[b], n), Array.from(raw(own[b][i], Uint16Array))))
  }
  // Attention. An output of either call is off by at most 2^-11 of itself and
  // 2^-10 of the largest value (weights and sums): together under 2^-8 of it.
  const vMax = Math.max(...Array.from(raw(cache.v, Uint16Array), (h) => Math.abs(half(h))))
  const near = (got, want) => {
    assert.strictEqual(got.length, want.length)
    for (let i = 0; i < got.length; i++) assert.ok(Math.abs(half(got[i]) - half(want[i])) <= vMax / 256, `${i}: ${half(got[i])} for ${half(want[i])}`)
  }
  const out = bytes(M * QD * 2)
  const out2 = bytes(M * QD * 2)
  const need = g.ops.pagedPrefillScratchBytes(cache, shape, M)
  g.ops.pagedAttnPrefill(q, M, shape, cache, rowStart, 0, 0, out, need ? bytes(need) : null)
  lens.forEach((n, b) => g.ops.attnPrefill(g.view(q, start[b] * QD * 4), n, shape, own[b][0], own[b][1], pos0, n, g.view(out2, start[b] * QD * 2)))
  near(raw(out, Uint16Array), raw(out2, Uint16Array))
  // one token a sequence: the prompts' last rows again, their weights added up
  const qLast = up(Float32Array.from([].concat(...lens.map((n, b) => Array.from(raw(q, Float32Array).subarray((start[b] + n - 1) * QD, (start[b] + n) * QD))))))
  const weights = bytes(2 * 64 * 4)
  const dec = bytes(2 * QD * 2)
  g.ops.pagedAttnDecode(qLast, shape, cache, 0, 0, weights, dec, bytes(g.ops.pagedDecodeScratchBytes(cache, shape, true)))
  const want = raw(out2, Uint16Array)
  near(raw(dec, Uint16Array), [].concat(...lens.map((n, b) => Array.from(want.subarray((start[b] + n - 1) * QD, (start[b] + n) * QD)))))
  const w = raw(weights, Float32Array)
  lens.forEach((n, b) => {
    const row = Array.from(w.subarray(64 * b, 64 * b + 64))
    assert.ok(row.slice(n).every((x) => x === 0) && row.slice(0, n).every((x) => x > 0))
    assert.ok(Math.abs(row.reduce((x, y) => x + y) - shape.heads) <= 1e-3)
  })
  // eviction to 18 entries, 2 first and 4 last ones protected
  const before = [raw(cache.k, Uint16Array), raw(cache.v, Uint16Array)]
  const to = Object.assign({}, cache, { table: up(Int32Array.from([1, 3, 6, 8])), ldTable: 2, lens: null })
  const toLens = bytes(8)
  const kept = bytes(2 * 18 * 4)
  const toWeights = bytes(2 * 18 * 4)
  const evictBytes = g.ops.pagedEvictScratchBytes(cache)
  g.ops.pagedEvict(cache, KVD, weights, 18, 2, 4, to, toLens, toWeights, kept, evictBytes ? bytes(evictBytes) : null)
  assert.deepStrictEqual(Array.from(raw(toLens, Int32Array)), [18, 18])
  const after = [raw(cache.k, Uint16Array), raw(cache.v, Uint16Array)]
  lens.forEach((n, b) => {
    const row = w.subarray(64 * b, 64 * b + n)
    const middle = Array.from({ length: n - 6 }, (_, i) => i + 2).sort((x, y) => row[y] - row[x] || x - y).slice(0, 12)
    const stay = [0, 1, ...middle.sort((x, y) => x - y), n - 4, n - 3, n - 2, n - 1]
    assert.deepStrictEqual(Array.from(raw(kept, Int32Array).subarray(18 * b, 18 * b + 18)), stay)
    assert.deepStrictEqual(Array.from(raw(toWeights, Float32Array).subarray(18 * b, 18 * b + 18)), stay.map((i) => row[i]))
    for (const i of [0, 1]) {
      const src = rowsOf(before[i], table[b], n)
      const dst = rowsOf(after[i], [[1, 3], [6, 8]][b], 18)
      assert.deepStrictEqual(dst, [].concat(...stay.map((e) => src.slice(e * KVD, (e + 1) * KVD))))
    }
  })
  // buffers smaller than the cache says are refused before any launch
  const small = bytes(16)
  invalid(() => g.ops.pagedAttnDecode(qLast, shape, Object.assign({}, cache, { k: small }), 0, 0, null, dec, small), 'k: ')
  invalid(() => g.ops.pagedAttnDecode(qLast, shape, Object.assign({}, cache, { table: small }), 0, 0, null, dec, small), 'table: ')
  invalid(() => g.ops.pagedAttnDecode(qLast, shape, cache, 0, 0, null, dec, small), 'scratch: ')
  invalid(() => g.ops.pagedAttnPrefill(q, M, shape, cache, small, 0, 0, small, null), 'out: ')
  invalid(() => g.ops.pagedHeadPrep(qkv, M, shape, null, null, tRope, ropeRows, small, cache, rowStart, q), 'pos: ')
  invalid(() => g.ops.pagedEvict(cache, KVD, weights, 18, 9, 10, to, toLens, null, kept, null), '9 sinks')
  assert.throws(() => g.ops.pagedAttnDecode(qLast, shape, Object.assign({}, cache, { lens: null }), 0, 0, null, dec, small), TypeError)
  g.dispose()
  return { kept: 36 }
}

const out = process.argv[2] === 'cpu' ? cpu() : gpu()
process.stdout.write(JSON.stringify(out) + '\n')
