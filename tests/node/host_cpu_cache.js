// Contracts of CacheAppendKernel, CacheAttentionKernel and DraftVerifyKernel
// without a GPU: descriptor checks and their messages, and fields with values
// that are none of theirs. Run by tests/test_node_cache.py.
"use strict";
const assert = require("assert");
const path = require("path");
const root = path.join(__dirname, "..", "..", "parakeet.wgsl_amd");
const host = require(path.join(root, "host"));
const addon = require(process.env.PK_NAPI_ADDON || path.join(root, "lib", "pk_napi.node"));

const MB = 1024 * 1024;
const arena = new host.GpuActivationArena({ createBuffer: ({ size }) => ({ address: BigInt(0x10000000), size }) }, 64 * MB);
function refused(fn, type, message) {
  assert.throws(fn, (e) => (e instanceof type && e.message.includes(message)) || assert.fail(`${e.name}: ${e.message}`));
}
let at = 0;
function slice(bytes) {
  at += MB;
  return arena.slice("s", at - MB, bytes);
}
const SIZES = [-1, 1000.5, 2 ** 32 + 1500, "1000", null, NaN];
const NUMBERS = ["0.5", null, true, BigInt(1), {}];

async function main() {
  const page = 2 * 16 * 64 * 2;
  const cache = {
    rowStarts: slice(16), lengths: slice(12), pageTable: slice(60), pagesPerSequence: 5, pages: 10, pageSize: 16,
    keys: slice(10 * page), values: slice(10 * page),
  };
  const rows = { rows: 11, sequences: 3, heads: 4, kvHeads: 2, headDim: 64, queries: slice(5632), cache };
  const append = Object.assign({
    label: "append", queryOutput: slice(5632), keys: slice(2816), values: slice(2816), rotaryDim: 64,
    rotary: "neighbours", frequencies: slice(128), positions: slice(44),
  }, rows);
  const attention = Object.assign({ label: "attention", output: slice(5632), window: 100, scale: 0.2, scoreCap: 30 }, rows);
  const verify = {
    label: "verify", rows: 11, sequences: 3, columns: 100, target: slice(2200), draft: slice(2200), temperature: 0.8,
    rowStarts: slice(16), tokens: slice(44), uniforms: slice(44), draws: slice(12), accepted: slice(12), nextTokens: slice(12),
  };
  const inCache = (change) => ({ cache: Object.assign({}, cache, change) });
  const kinds = [
    [host.CacheAppendKernel, append, "cacheAppend", ["queryStride", "queryOutputStride", "keyStride", "valueStride"], [], [
      [{ rotary: "thirds" }, Error, "append has an unsupported rotary kind thirds"],
      [{ rotaryDim: 66 }, RangeError, "append rotary dim must be even and at most 64"],
      [{ frequencies: undefined }, Error, "append needs frequencies with a rotary dim, and only then"],
      [{ queryOutput: undefined }, Error, "append needs queries and a query output with heads, and only then"],
      [{ queryOutput: append.keys }, RangeError, "append query output needs 5632 bytes; arena slice has 2816"],
      [inCache({ pageStride: -8 }), RangeError, "append pageStride must be a non-negative integer"],
      [inCache({ pageStride: 4100 }), RangeError, "append page stride must be a multiple of 8 of at least a page"],
      [inCache({ pages: 11 }), RangeError, "append key cache needs 45056 bytes; arena slice has 40960"],
      [inCache({ lengths: undefined }), Error, "append needs row starts, lengths, a page table and caches"],
      [{ cache: undefined }, Error, "cache append descriptor is missing a required field"],
    ]],
    [host.CacheAttentionKernel, attention, "cacheAttention", ["queryStride", "outputStride"], ["scale", "scoreCap"], [
      [{ causal: 1 }, Error, "attention causal must be a boolean"],
      [{ causal: false }, Error, "attention has a window without causal"],
      [{ heads: 3 }, RangeError, "attention heads must be a multiple of the 2 kv heads"],
      [{ scoreCap: -1 }, RangeError, "attention score cap must be 0 or in [2^-20, 2^20]"],
      [{ output: attention.queries }, Error, "attention output must not overlap queries"],
      [inCache({ pageSize: 0 }), RangeError, "Invalid cache pages [10 of 0, 5 of a sequence] for attention"],
    ]],
    [host.DraftVerifyKernel, verify, "verify", ["targetStride", "draftStride"], ["temperature"], [
      [{ mode: "beam" }, Error, "verify has an unsupported mode beam"],
      [{ draws: undefined }, Error, "verify needs uniforms and draws"],
      [{ accepted: verify.nextTokens }, Error, "verify outputs must not overlap each other or the inputs"],
      [{ rows: 12 }, RangeError, "verify target needs 2400 bytes; arena slice has 2200"],
    ]],
  ];
  for (const [Kernel, base, prefix, sizes, numbers, cases] of kinds) {
    const kernel = await Kernel.create({}, arena), { label } = base;
    const make = (change) => Object.assign({}, base, change);
    kernel.validateDescriptor(make());
    for (const [change, type, message] of cases) refused(() => kernel.validateDescriptor(make(change)), type, message);
    for (const name of sizes)
      for (const value of SIZES)
        refused(() => kernel.validateDescriptor(make({ [name]: value })), RangeError, `${label} ${name} must be a non-negative 32-bit integer`);
    for (const name of numbers)
      for (const value of NUMBERS)
        refused(() => kernel.validateDescriptor(make({ [name]: value })), Error, `${label} ${name} must be a number`);
    // the addon by itself
    const validate = addon[`${prefix}Validate`], plain = () => kernel.nativeDescriptor(make());
    validate(plain());
    for (const name of sizes)
      for (const value of SIZES.filter((v) => v !== null).concat([true, {}]))
        refused(() => validate(Object.assign(plain(), { [name]: value })), Error, `${name} must be a non-negative 32-bit integer`);
    for (const name of numbers)
      for (const value of NUMBERS.filter((v) => v !== null))
        refused(() => validate(Object.assign(plain(), { [name]: value })), Error, `${name} must be a number`);
    for (const name of Object.keys(plain()).filter((n) => n.endsWith("Bytes"))) {
      const binding = name.slice(0, -5);
      refused(() => validate(Object.assign(plain(), { [binding]: "buffer" })), Error, `${binding} must be a device pointer`);
      refused(() => validate(Object.assign(plain(), { [name]: -4 })), Error, `${name} must be a byte count`);
    }
    if (prefix !== "verify")
      for (const value of [-8, 1.5, "64", {}])
        refused(() => validate(Object.assign(plain(), { pageStride: value })), Error, "pageStride must be a non-negative integer");
    kernel.destroy();
    refused(() => kernel.createDispatch(make()), Error, "kernel was destroyed");
  }
  const greedy = await host.DraftVerifyKernel.create({}, arena);
  greedy.validateDescriptor(Object.assign({}, verify, { mode: "greedy", draft: undefined, uniforms: undefined, draws: undefined }));
  assert.strictEqual(host.CACHE_NO_PAGE, 0xffffffff);
  assert.strictEqual(host.VERIFY_NO_TOKEN, 0xffffffff);
  console.log("host_cpu_cache ok");
}
main().catch((e) => { console.error(e); process.exit(1); });
